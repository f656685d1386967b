"""A paged key / value cache held in 4 bits, and the decode that reads it.

``Int4KVCache`` owns the pool; ``append_kv_int4`` writes a prompt's or a decode
step's rows, ``paged_attention_int4`` is the decode (``paged_attention`` over
this cache), and ``read_kv_int4`` returns rows as the values they stand for (the
cached context of a prompt's next chunk, for ``prompt_attention``).  No
counterpart in the reference, whose caches hold 16-bit rows (paged.py:22-23).
"""

import ctypes
import math

import torch

from flagattention_b200 import _lib
from flagattention_b200._torch import ptr, require_cuda, status_word, stream_of


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
        size = ctypes.c_int64(0)
        _lib.check(_lib.lib().fa_kv4_cache_bytes(ctypes.byref(self._struct(None)),
                                                 ctypes.byref(size)), "fa_kv4_cache_bytes")
        tiles = self.block_size // 16
        row = self.head_size + 8 * (self.head_size // self.group_size)
        self.data = torch.zeros((self.num_blocks, self.num_kv_heads, tiles, 16 * row),
                                dtype=torch.uint8, device=device)
        assert self.data.numel() == size.value

    @property
    def device(self):
        return self.data.device

    def _struct(self, data):
        code = _lib.FA_DTYPE_F16 if self.dtype == torch.float16 else _lib.FA_DTYPE_BF16
        return _lib.Kv4Cache(data, self.num_blocks, self.num_kv_heads, self.block_size,
                             self.head_size, self.group_size, code)

    def struct(self):
        return self._struct(self.data.data_ptr())


def _rows16(x):
    """x, or a contiguous copy where the kernels cannot address its rows."""
    if x.stride(-1) == 1 and all(s % 8 == 0 for s in x.stride()[:-1]) and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _check_slots(slot_mapping, cache):
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1:
        raise _lib.InvalidArgument("slot_mapping must be int64 [n]")
    if slot_mapping.device != cache.device:
        raise _lib.InvalidArgument("all tensors must be on the cache's device")
    return slot_mapping.contiguous()


def append_kv_int4(k, v, cache, slot_mapping):
    """Write rows k, v [n, num_kv_heads, head_size] (cache.dtype) to the pool
    slots ``block * block_size + offset`` of slot_mapping (int64 [n]), in place;
    returns the cache.  A slot outside the pool (negative: padding) skips its
    row; slots must be distinct.  A group of dims that holds a NaN or an
    infinity reads back as NaN."""
    require_cuda(k, v, slot_mapping)
    want = (slot_mapping.shape[0] if slot_mapping.dim() else -1, cache.num_kv_heads,
            cache.head_size)
    if tuple(k.shape) != want or tuple(v.shape) != want:
        raise _lib.InvalidArgument(f"k and v must be [n, {want[1]}, {want[2]}]")
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise _lib.InvalidArgument(f"rows must be in the cache's dtype ({cache.dtype})")
    slot_mapping = _check_slots(slot_mapping, cache)
    if k.device != cache.device or v.device != cache.device:
        raise _lib.InvalidArgument("all tensors must be on the cache's device")
    k, v = _rows16(k), _rows16(v)
    _lib.check(_lib.lib().fa_kv4_append(ctypes.byref(cache.struct()), ptr(k), k.stride(0),
                                        k.stride(1), ptr(v), v.stride(0), v.stride(1),
                                        ptr(slot_mapping), k.shape[0], stream_of(k)),
               "fa_kv4_append")
    return cache


def read_kv_int4(cache, slot_mapping):
    """(k, v) [n, num_kv_heads, head_size] of the pool slots in slot_mapping
    (int64 [n]), as the values their codes stand for, in cache.dtype; zeros for
    a slot outside the pool."""
    require_cuda(slot_mapping)
    slot_mapping = _check_slots(slot_mapping, cache)
    shape = (slot_mapping.shape[0], cache.num_kv_heads, cache.head_size)
    k = torch.empty(shape, dtype=cache.dtype, device=cache.device)
    v = torch.empty(shape, dtype=cache.dtype, device=cache.device)
    _lib.check(_lib.lib().fa_kv4_read(ctypes.byref(cache.struct()), ptr(k), k.stride(0),
                                      k.stride(1), ptr(v), v.stride(0), v.stride(1),
                                      ptr(slot_mapping), shape[0], stream_of(k)),
               "fa_kv4_read")
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
    require_cuda(query, context_lens, block_tables)
    if query.dim() != 3 or query.shape[2] != cache.head_size:
        raise _lib.InvalidArgument("query must be [num_seqs, num_q_heads, head_size of the cache]")
    if query.dtype != cache.dtype:
        raise _lib.InvalidArgument(f"the query must be in the cache's dtype ({cache.dtype})")
    num_seqs, hq, d = query.shape
    if hq == 0 or hq % cache.num_kv_heads != 0:
        raise _lib.InvalidArgument("num_q_heads must be a multiple of the cache's kv heads")
    if context_lens.dtype != torch.int32 or block_tables.dtype != torch.int32:
        raise _lib.InvalidArgument("context_lens and block_tables must be int32")
    if tuple(context_lens.shape) != (num_seqs,) or block_tables.dim() != 2 or \
            block_tables.shape[0] != num_seqs:
        raise _lib.InvalidArgument("context_lens [num_seqs] and block_tables [num_seqs, width]")
    if any(t.device != cache.device for t in (query, context_lens, block_tables)):
        raise _lib.InvalidArgument("all tensors must be on the cache's device")
    query, context_lens = _rows16(query), context_lens.contiguous()
    if block_tables.stride(-1) != 1:
        block_tables = block_tables.contiguous()
    out = torch.empty((num_seqs, hq, d), dtype=query.dtype, device=query.device)
    lse = torch.empty((num_seqs, hq), dtype=torch.float32, device=query.device) \
        if return_lse else None
    a = _lib.Kv4AttentionArgs()
    a.q, a.q_stride_b, a.q_stride_h = query.data_ptr(), query.stride(0), query.stride(1)
    a.cache = cache.struct()
    a.block_table, a.bt_stride = block_tables.data_ptr(), block_tables.stride(0)
    a.bt_width = block_tables.shape[1]
    a.seq_lens = context_lens.data_ptr()
    a.batch, a.num_q_heads = num_seqs, hq
    a.scale = float(attn_scale if attn_scale is not None else 1.0 / math.sqrt(d))
    a.o, a.o_stride_b, a.o_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    a.lse = lse.data_ptr() if return_lse else None
    a.status = status_word(query.device).data_ptr()
    po, pl, mg = (ctypes.c_size_t(0) for _ in range(3))
    _lib.check(_lib.lib().fa_kv4_attention_workspace_size(
        ctypes.byref(a), ctypes.byref(po), ctypes.byref(pl), ctypes.byref(mg)),
        "fa_kv4_attention_workspace_size")
    ws = torch.empty(po.value + pl.value + mg.value, dtype=torch.uint8, device=query.device)
    a.part_o = ws.data_ptr()
    a.part_lse = a.part_o + po.value
    a.merge = a.part_lse + pl.value
    _lib.check(_lib.lib().fa_kv4_attention(ctypes.byref(a), stream_of(query)), "fa_kv4_attention")
    return (out, lse) if return_lse else out
