"""Attention over whole prompts: packed sequences of different lengths.

``prompt_attention`` is the step before the decode: every token of a prompt
attends to the tokens up to its own (and to ``lk - lq`` earlier keys when the
sequence has more keys than new tokens, as the next chunk of a long prompt
does).  The mathematics is the forward of ``flag_attn.flash_attention``
(flash.py:269, bottom-right causal mask as in split_kv.py:88-92); packing
several lengths in one call has no counterpart in the reference.  Forward
only, as every operator of this package.
"""

import ctypes
import functools
import math

import torch

from flagattention_b200 import _lib
from flagattention_b200._torch import (current_device, dtype_code, empty, launch_lock, raw_stream,
                                       require_cuda, status_ptr, stream_workspace)


_pack, _args = _lib.packer(_lib.PromptArgs)


def _rows(x):
    """(x, address, token stride, head stride): x, or a contiguous copy where the
    kernel cannot address its rows (inner stride, broadcast dims, 16-byte
    alignment)."""
    t, h, d = x.stride()
    p = x.data_ptr()
    if d != 1 or not t or not h or (t | h | (p >> 1)) & 7:
        x = x.clone(memory_format=torch.contiguous_format)
        t, h, _ = x.stride()
        p = x.data_ptr()
    return x, p, t, h


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device_index, batch, total_q, total_k, hq, hk, d_v, causal):
    """Scratch of a call of these sizes on this (the current) device."""
    a = _lib.PromptArgs(batch=batch, total_q=total_q, total_k=total_k, num_q_heads=hq,
                        num_kv_heads=hk, d_v=d_v, causal=causal)
    size = ctypes.c_size_t(0)
    _lib.check(_lib.lib().fa_prompt_workspace_size(ctypes.byref(a), ctypes.byref(size)),
               "fa_prompt_workspace_size")
    return size.value


def prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, causal=True, sm_scale=None,
                     return_lse=False):
    """Attention of packed prompts.

    q: [total_q, Hq, D]; k: [total_k, Hk, D]; v: [total_k, Hk, Dv], bf16 or
    f16, Hq a multiple of Hk (at most 128 query heads per kv head), head sizes
    multiples of 8 up to D = 192, Dv = 128.  cu_seqlens_q / cu_seqlens_k:
    int32 [batch + 1] on the GPU, starting at 0: sequence b owns rows
    cu[b] .. cu[b + 1] - 1 (cu_seqlens_k defaults to cu_seqlens_q).  Causal
    masking is bottom-right aligned: query i of lq sees keys 0 .. lk - lq + i.
    Returns out [total_q, Hq, Dv]; with return_lse also the log-sum-exp of
    the scaled scores, f32 [Hq, total_q].  A row that sees no key gets zeros
    and -inf; rows past cu_seqlens_q[-1] are not written.  Keys and values that
    a row does not see do not reach it, whatever they hold; a NaN or an infinity
    in a value that it sees makes that element of the row NaN or infinite.
    """
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    dev = q.get_device()
    if dev < 0 or k.get_device() != dev or v.get_device() != dev or \
            cu_seqlens_q.get_device() != dev or cu_seqlens_k.get_device() != dev:
        require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k)
        raise _lib.InvalidArgument("all tensors must be on one device")
    if dev != current_device():
        with torch.cuda.device(dev):
            return prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, sm_scale,
                                    return_lse)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise _lib.InvalidArgument("q, k, v must be [tokens, heads, head size]")
    (total_q, hq, d), (total_k, hk, d_k), (total_v, hv, d_v) = q.shape, k.shape, v.shape
    if d_k != d or total_v != total_k or hv != hk:
        raise _lib.InvalidArgument("q/k/v shapes disagree")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise _lib.InvalidArgument("q, k and v dtypes differ")
    if hk == 0 or hq == 0 or hq % hk != 0:
        raise _lib.InvalidArgument("number of heads in q must be a multiple of that in k & v")
    if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_k.dtype != torch.int32 or \
            cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] < 1 or \
            cu_seqlens_k.shape != cu_seqlens_q.shape:
        raise _lib.InvalidArgument("cu_seqlens must be int32 [batch + 1]")
    code = dtype_code(q)
    batch = cu_seqlens_q.shape[0] - 1
    causal = 1 if causal else 0
    (q_t, q_h, q_d), (k_t, k_h, k_d), (v_t, v_h, v_d) = q.stride(), k.stride(), v.stride()
    q_p, k_p, v_p = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not (q_d == k_d == v_d == 1 and q_t and q_h and k_t and k_h and v_t and v_h) or \
            (q_t | q_h | k_t | k_h | v_t | v_h | (q_p | k_p | v_p) >> 1) & 7:
        (q, q_p, q_t, q_h), (k, k_p, k_t, k_h), (v, v_p, v_t, v_h) = _rows(q), _rows(k), _rows(v)
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    out = empty((total_q, hq, d_v), dtype, dev)
    lse = empty((hq, total_q), torch.float32, dev) if return_lse else None
    size = _workspace_bytes(dev, batch, total_q, total_k, hq, hk, d_v, causal) \
        if hq // hk <= 128 and 0 < d_v <= 128 else 0
    stream = raw_stream(dev)
    with launch_lock:
        ws, base = stream_workspace(size, dev, stream) if size else (None, 0)
        # field order of fa_prompt_args
        _pack(q_p, q_t, q_h, k_p, k_t, k_h, v_p, v_t, v_h,
              cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
              batch, total_q, total_k, hq, hk, d, d_v, causal, code,
              1.0 / math.sqrt(d) if sm_scale is None else sm_scale,
              out.data_ptr(), hq * d_v, d_v, lse.data_ptr() if return_lse else 0,
              base, status_ptr(dev))
        st = _lib.lib().fa_prompt_attention(_args, stream)
    if st:
        _lib.check(st, "fa_prompt_attention")
    return (out, lse) if return_lse else out
