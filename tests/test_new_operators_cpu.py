"""Argument checks of the prompt and 4-bit cache entry points, which run before
any CUDA call (the pointers below are never dereferenced), and the documented
layout of a cache tile as a bijection."""

import ctypes

import pytest

import flagattention_b200 as fa
from flagattention_b200 import _lib

FAKE = 1 << 20


def prompt_args(**over):
    a = _lib.PromptArgs(q=FAKE, q_stride_t=1024, q_stride_h=128, k=FAKE, k_stride_t=256,
                        k_stride_h=128, v=FAKE, v_stride_t=256, v_stride_h=128, cu_q=FAKE,
                        cu_k=FAKE, batch=2, total_q=10, total_k=10, num_q_heads=8, num_kv_heads=2,
                        d_qk=128, d_v=128, causal=1, dtype=0, scale=0.1, o=FAKE, o_stride_t=1024,
                        o_stride_h=128)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, want", [
    (dict(batch=-1), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(num_q_heads=9), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(num_q_heads=516, num_kv_heads=4), _lib.FA_ERR_UNSUPPORTED),
    (dict(dtype=2), _lib.FA_ERR_UNSUPPORTED),
    (dict(d_qk=200), _lib.FA_ERR_UNSUPPORTED),
    (dict(d_v=136), _lib.FA_ERR_UNSUPPORTED),
    (dict(d_qk=100), _lib.FA_ERR_UNSUPPORTED),
    (dict(scale=0.0), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(scale=float("nan")), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(scale=float("inf")), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(q=None), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(cu_k=None), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(k=FAKE + 2), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(q_stride_h=132), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(batch=0), _lib.FA_OK),
    (dict(total_q=0), _lib.FA_OK),
])
def test_prompt_arguments(over, want):
    assert _lib.lib().fa_prompt_attention(ctypes.byref(prompt_args(**over)), None) == want


def test_prompt_null_arguments():
    lib = _lib.lib()
    assert lib.fa_prompt_attention(None, None) == _lib.FA_ERR_INVALID_ARGUMENT
    assert lib.fa_prompt_workspace_size(None, None) == _lib.FA_ERR_INVALID_ARGUMENT


def cache_struct(**over):
    c = _lib.Kv4Cache(FAKE, 4, 2, 16, 128, 64, 0)
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("over, want", [
    (dict(), 4 * 2 * 16 * 144),
    (dict(head_size=64, group_size=32), 4 * 2 * 16 * 80),
    (dict(head_size=256, group_size=128, block_size=48), 4 * 2 * 48 * 272),
    (dict(num_blocks=0), 0),
])
def test_cache_bytes(over, want):
    n = ctypes.c_int64(-1)
    assert _lib.lib().fa_kv4_cache_bytes(ctypes.byref(cache_struct(**over)), ctypes.byref(n)) == 0
    assert n.value == want


@pytest.mark.parametrize("over, want", [
    (dict(head_size=96), _lib.FA_ERR_UNSUPPORTED), (dict(group_size=16), _lib.FA_ERR_UNSUPPORTED),
    (dict(head_size=64, group_size=128), _lib.FA_ERR_UNSUPPORTED),
    (dict(head_size=256, group_size=32), _lib.FA_ERR_UNSUPPORTED),
    (dict(block_size=20), _lib.FA_ERR_UNSUPPORTED), (dict(dtype=2), _lib.FA_ERR_UNSUPPORTED),
    (dict(num_kv_heads=0), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(num_blocks=-1), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(data=FAKE + 8), _lib.FA_ERR_INVALID_ARGUMENT),
    (dict(num_blocks=2 ** 30, num_kv_heads=8), _lib.FA_ERR_UNSUPPORTED),
])
def test_cache_refused(over, want):
    lib, c = _lib.lib(), cache_struct(**over)
    n = ctypes.c_int64()
    assert lib.fa_kv4_cache_bytes(ctypes.byref(c), ctypes.byref(n)) == want
    assert lib.fa_kv4_append(ctypes.byref(c), FAKE, 256, 128, FAKE, 256, 128, FAKE, 1, None) == want
    assert lib.fa_kv4_read(ctypes.byref(c), FAKE, 256, 128, FAKE, 256, 128, FAKE, 1, None) == want
    a = _lib.Kv4AttentionArgs(q=FAKE, cache=c, batch=1, num_q_heads=8, scale=0.1)
    assert lib.fa_kv4_attention(ctypes.byref(a), None) == want


def test_rows_and_attention_refused():
    lib, c = _lib.lib(), cache_struct()
    bad = _lib.FA_ERR_INVALID_ARGUMENT
    call = lambda *a: lib.fa_kv4_append(ctypes.byref(c), *a, None)  # noqa: E731
    assert call(FAKE, 256, 128, FAKE, 256, 128, FAKE, -1) == bad
    assert call(None, 256, 128, FAKE, 256, 128, FAKE, 1) == bad
    assert call(FAKE + 2, 256, 128, FAKE, 256, 128, FAKE, 1) == bad
    assert call(FAKE, 257, 128, FAKE, 256, 128, FAKE, 1) == bad
    assert call(FAKE, 256, 128, FAKE, 256, 128, FAKE + 4, 1) == bad
    assert call(None, 256, 128, None, 256, 128, None, 0) == _lib.FA_OK      # nothing to write
    a = _lib.Kv4AttentionArgs(q=FAKE, cache=c, batch=1, num_q_heads=8, scale=0.1)
    for over in (dict(num_q_heads=7), dict(scale=-1.0), dict(bt_width=-1), dict(seq_lens=None)):
        b = _lib.Kv4AttentionArgs.from_buffer_copy(a)
        for k, v in over.items():
            setattr(b, k, v)
        assert lib.fa_kv4_attention(ctypes.byref(b), None) == bad
    b = _lib.Kv4AttentionArgs.from_buffer_copy(a)
    b.batch = 0
    assert lib.fa_kv4_attention(ctypes.byref(b), None) == _lib.FA_OK


def test_cache_needs_a_gpu():
    with pytest.raises(fa.InvalidArgument):
        fa.Int4KVCache(2, 2, 16, 128, device="cpu")
    with pytest.raises(fa.Unsupported):
        fa.Int4KVCache(2, 2, 16, 96)
    import torch
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(fa.InvalidArgument):
        fa.prompt_attention(x, x, x, torch.tensor([0, 4], dtype=torch.int32))
