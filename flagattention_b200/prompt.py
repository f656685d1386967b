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
import math

import torch

from flagattention_b200 import _lib
from flagattention_b200._torch import dtype_code, require_cuda, status_word, stream_of


def _rows16(x):
    """x, or a contiguous copy where the kernel cannot address its rows
    (inner stride, 16-byte alignment)."""
    if x.stride(-1) == 1 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0 and \
            x.stride(0) >= 0 and x.stride(1) >= 0 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


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
    and -inf; rows past cu_seqlens_q[-1] are not written.
    """
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise _lib.InvalidArgument("q, k, v must be [tokens, heads, head size]")
    (total_q, hq, d), (total_k, hk, _), d_v = q.shape, k.shape, v.shape[2]
    if k.shape[2] != d or v.shape[:2] != k.shape[:2]:
        raise _lib.InvalidArgument("q/k/v shapes disagree")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise _lib.InvalidArgument("q, k and v dtypes differ")
    if hk == 0 or hq == 0 or hq % hk != 0:
        raise _lib.InvalidArgument("number of heads in q must be a multiple of that in k & v")
    for cu in (cu_seqlens_q, cu_seqlens_k):
        if cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 1 or \
                cu.shape != cu_seqlens_q.shape:
            raise _lib.InvalidArgument("cu_seqlens must be int32 [batch + 1]")
    devices = {t.device for t in (q, k, v, cu_seqlens_q, cu_seqlens_k)}
    if len(devices) != 1:
        raise _lib.InvalidArgument("all tensors must be on one device")
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    out = torch.empty((total_q, hq, d_v), dtype=q.dtype, device=q.device)
    lse = torch.empty((hq, total_q), dtype=torch.float32, device=q.device) if return_lse else None
    a = _lib.PromptArgs()
    a.q, a.q_stride_t, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    a.k, a.k_stride_t, a.k_stride_h = k.data_ptr(), k.stride(0), k.stride(1)
    a.v, a.v_stride_t, a.v_stride_h = v.data_ptr(), v.stride(0), v.stride(1)
    a.cu_q, a.cu_k = cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr()
    a.batch, a.total_q, a.total_k = cu_seqlens_q.shape[0] - 1, total_q, total_k
    a.num_q_heads, a.num_kv_heads, a.d_qk, a.d_v = hq, hk, d, d_v
    a.causal = int(bool(causal))
    a.dtype = dtype_code(q)
    a.scale = float(sm_scale if sm_scale is not None else 1.0 / math.sqrt(d))
    a.o, a.o_stride_t, a.o_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    a.lse = lse.data_ptr() if return_lse else None
    a.status = status_word(q.device).data_ptr()
    _lib.check(_lib.lib().fa_prompt_attention(ctypes.byref(a), stream_of(q)),
               "fa_prompt_attention")
    return (out, lse) if return_lse else out
