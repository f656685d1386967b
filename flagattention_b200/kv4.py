"""A paged key / value cache held in 4 bits, and the decode that reads it.

``Int4KVCache`` owns the pool; ``append_kv_int4`` writes a prompt's or a decode
step's rows, ``paged_attention_int4`` is the decode (``paged_attention`` over
this cache), and ``read_kv_int4`` returns rows as the values they stand for (the
cached context of a prompt's next chunk, for ``prompt_attention``).  No
counterpart in the reference, whose caches hold 16-bit rows (paged.py:22-23).
"""

import ctypes
import functools
import math

import torch

from flagattention_b200 import _lib
from flagattention_b200._torch import (current_device, empty, launch_lock, raw_stream,
                                       require_cuda, stream_workspace)


_pack_attention, _attention_args = _lib.packer(_lib.Kv4AttentionArgs)


class Int4KVCache:
    """Pool of num_blocks blocks of block_size tokens, num_kv_heads heads of
    head_size dims (64, 128 or 256), keys and values.

    Groups of group_size dims (32, 64 or 128; one to four per head) share a
    minimum and a scale in ``dtype`` (bf16 or f16, the type of the rows written,
    read and queried): D + 8 D / group_size bytes per token and head instead of
    4 D.  block_size must be a multiple of 16.  ``data`` is the pool, uint8
    [num_blocks, num_kv_heads, block_size // 16, bytes of 16 tokens] (layout in
    csrc/kv4.cuh), zeros at first (every value 0).
    """

    def __init__(self, num_blocks, num_kv_heads, block_size, head_size, dtype=torch.bfloat16,
                 group_size=64, device="cuda"):
        self.num_blocks, self.num_kv_heads = int(num_blocks), int(num_kv_heads)
        self.block_size, self.head_size = int(block_size), int(head_size)
        self.dtype, self.group_size = dtype, int(group_size)
        if dtype not in (torch.bfloat16, torch.float16):
            raise _lib.Unsupported("a 4-bit cache takes bf16 or f16 rows")
        device = torch.device(device)
        if device.type != "cuda":
            raise _lib.InvalidArgument("flagattention_b200 operators take CUDA tensors only "
                                       "(there is no CPU path)")
        self.dtype_code = _lib.FA_DTYPE_F16 if dtype == torch.float16 else _lib.FA_DTYPE_BF16
        self._struct = _lib.Kv4Cache(None, self.num_blocks, self.num_kv_heads, self.block_size,
                                     self.head_size, self.group_size, self.dtype_code)
        size = ctypes.c_int64(0)
        _lib.check(_lib.lib().fa_kv4_cache_bytes(ctypes.byref(self._struct), ctypes.byref(size)),
                   "fa_kv4_cache_bytes")
        tiles = self.block_size // 16
        row = self.head_size + 8 * (self.head_size // self.group_size)
        self.data = torch.zeros((self.num_blocks, self.num_kv_heads, tiles, 16 * row),
                                dtype=torch.uint8, device=device)
        assert self.data.numel() == size.value

    @property
    def device(self):
        return self.data.device

    def fields(self):
        """The values of the library's ``fa_kv4_cache``, in order."""
        return (self.data.data_ptr(), self.num_blocks, self.num_kv_heads, self.block_size,
                self.head_size, self.group_size, self.dtype_code)

    def struct(self):
        """The pool as the library's ``fa_kv4_cache``."""
        self._struct.data = self.data.data_ptr()
        return self._struct


def _rows16(x):
    """x, or a contiguous copy where the kernels cannot address its rows."""
    t, h, d = x.stride()
    if d == 1 and t and h and not (t | h | (x.data_ptr() >> 1)) & 7:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _check_slots(slot_mapping, cache):
    if not slot_mapping.is_cuda:
        require_cuda(slot_mapping)
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1:
        raise _lib.InvalidArgument("slot_mapping must be int64 [n]")
    if slot_mapping.get_device() != cache.data.get_device():
        raise _lib.InvalidArgument("all tensors must be on the cache's device")
    return slot_mapping.contiguous()


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index, batch, hq, hk, head_size, group_size, dtype):
    """(part_o, part_lse, merge) bytes for these sizes on this (the current) device."""
    a = _lib.Kv4AttentionArgs()
    a.cache = _lib.Kv4Cache(None, 0, hk, 16, head_size, group_size, dtype)
    a.batch, a.num_q_heads, a.scale = batch, hq, 1.0
    po, pl, mg = (ctypes.c_size_t(0) for _ in range(3))
    _lib.check(_lib.lib().fa_kv4_attention_workspace_size(
        ctypes.byref(a), ctypes.byref(po), ctypes.byref(pl), ctypes.byref(mg)),
        "fa_kv4_attention_workspace_size")
    return po.value, pl.value, mg.value


def append_kv_int4(k, v, cache, slot_mapping):
    """Write rows k, v [n, num_kv_heads, head_size] (cache.dtype) to the pool
    slots ``block * block_size + offset`` of slot_mapping (int64 [n]), in place;
    returns the cache.  A slot outside the pool (negative: padding) skips its
    row; slots must be distinct.  A group of dims that holds a NaN or an
    infinity reads back as NaN."""
    if not (k.is_cuda and v.is_cuda):
        require_cuda(k, v)
    slot_mapping = _check_slots(slot_mapping, cache)
    n = slot_mapping.shape[0]
    want = (n, cache.num_kv_heads, cache.head_size)
    if k.shape != want or v.shape != want:
        raise _lib.InvalidArgument(f"k and v must be [n, {want[1]}, {want[2]}]")
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise _lib.InvalidArgument(f"rows must be in the cache's dtype ({cache.dtype})")
    dev = slot_mapping.get_device()
    if k.get_device() != dev or v.get_device() != dev:
        raise _lib.InvalidArgument("all tensors must be on the cache's device")
    if dev != current_device():
        with torch.cuda.device(dev):
            return append_kv_int4(k, v, cache, slot_mapping)
    k, v = _rows16(k), _rows16(v)
    (k_t, k_h, _), (v_t, v_h, _) = k.stride(), v.stride()
    st = _lib.lib().fa_kv4_append(ctypes.byref(cache.struct()), k.data_ptr(), k_t, k_h,
                                  v.data_ptr(), v_t, v_h, slot_mapping.data_ptr(), n,
                                  raw_stream(dev))
    if st:
        _lib.check(st, "fa_kv4_append")
    return cache


def read_kv_int4(cache, slot_mapping):
    """(k, v) [n, num_kv_heads, head_size] of the pool slots in slot_mapping
    (int64 [n]), as the values their codes stand for, in cache.dtype; zeros for
    a slot outside the pool."""
    slot_mapping = _check_slots(slot_mapping, cache)
    n, heads, d = slot_mapping.shape[0], cache.num_kv_heads, cache.head_size
    dev = slot_mapping.get_device()
    if dev != current_device():
        with torch.cuda.device(dev):
            return read_kv_int4(cache, slot_mapping)
    k, v = empty((n, heads, d), cache.dtype, dev), empty((n, heads, d), cache.dtype, dev)
    st = _lib.lib().fa_kv4_read(ctypes.byref(cache.struct()), k.data_ptr(), heads * d, d,
                                v.data_ptr(), heads * d, d, slot_mapping.data_ptr(), n,
                                raw_stream(dev))
    if st:
        _lib.check(st, "fa_kv4_read")
    return k, v


def paged_attention_int4(query, cache, context_lens, block_tables, attn_scale=None,
                         return_lse=False):
    """``paged_attention`` (paged.py:20) over a 4-bit cache.

    query: [num_seqs, num_q_heads, head_size] in cache.dtype; context_lens:
    int32 [num_seqs]; block_tables: int32 [num_seqs, max blocks].  attn_scale
    defaults to head_size ** -0.5.  Returns out like the query, with return_lse
    also the log-sum-exp f32 [num_seqs, num_q_heads].  A sequence without
    cached tokens gets zeros and -inf.
    """
    dev = query.get_device()
    if dev < 0 or cache.data.get_device() != dev or context_lens.get_device() != dev or \
            block_tables.get_device() != dev:
        require_cuda(query, context_lens, block_tables)
        raise _lib.InvalidArgument("all tensors must be on the cache's device")
    if dev != current_device():
        with torch.cuda.device(dev):
            return paged_attention_int4(query, cache, context_lens, block_tables, attn_scale,
                                        return_lse)
    if query.dim() != 3 or query.shape[2] != cache.head_size:
        raise _lib.InvalidArgument("query must be [num_seqs, num_q_heads, head_size of the cache]")
    c_dtype = cache.dtype
    if query.dtype != c_dtype:
        raise _lib.InvalidArgument(f"the query must be in the cache's dtype ({cache.dtype})")
    num_seqs, hq, d = query.shape
    if hq == 0 or hq % cache.num_kv_heads != 0:
        raise _lib.InvalidArgument("num_q_heads must be a multiple of the cache's kv heads")
    if context_lens.dtype != torch.int32 or block_tables.dtype != torch.int32:
        raise _lib.InvalidArgument("context_lens and block_tables must be int32")
    if context_lens.shape != (num_seqs,) or block_tables.dim() != 2 or \
            block_tables.shape[0] != num_seqs:
        raise _lib.InvalidArgument("context_lens [num_seqs] and block_tables [num_seqs, width]")
    query, context_lens = _rows16(query), context_lens.contiguous()
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    out = empty((num_seqs, hq, d), c_dtype, dev)
    lse = empty((num_seqs, hq), torch.float32, dev) if return_lse else None
    po, pl, mg = _workspace_bytes(dev, num_seqs, hq, cache.num_kv_heads, d, cache.group_size,
                                  cache.dtype_code)
    stream = raw_stream(dev)
    q_b, q_h, _ = query.stride()
    with launch_lock:
        ws, base = stream_workspace(po + pl + mg, dev, stream)
        # field order of fa_kv4_attention_args
        _pack_attention(query.data_ptr(), q_b, q_h, *cache.fields(), block_tables.data_ptr(),
                        block_tables.stride(0), block_tables.shape[1], context_lens.data_ptr(),
                        num_seqs, hq, 1.0 / math.sqrt(d) if attn_scale is None else attn_scale,
                        out.data_ptr(), hq * d, d, lse.data_ptr() if return_lse else 0,
                        base, base + po, base + po + pl)
        st = _lib.lib().fa_kv4_attention(_attention_args, stream)
    if st:
        _lib.check(st, "fa_kv4_attention")
    return (out, lse) if return_lse else out
