"""Calls made while another device is current launch on their tensors' device.

One GPU is enough: the current device is a number that the tests keep, and
entering a device changes only that number, so nothing runs anywhere else.
"""

import pytest
import torch

import flagattention_b200 as fa
from flagattention_b200 import _torch, kv4, mla, paged, prompt, split_kv

pytestmark = pytest.mark.gpu


class Launches(list):
    pass


@pytest.fixture
def elsewhere(monkeypatch):
    """Device 1 is current; returns the devices that were current at each launch."""
    now, launches = [1], Launches()
    launches.now = now

    class Entered:
        def __init__(self, device):
            if device is None:
                device = now[-1]
            self.device = device if isinstance(device, int) else device.index

        def __enter__(self):
            now.append(self.device)

        def __exit__(self, *_):
            now.pop()

    raw_stream = _torch.raw_stream
    monkeypatch.setattr(torch.cuda, "device", Entered)
    for module in (kv4, prompt):
        monkeypatch.setattr(module, "current_device", lambda: now[-1], raising=False)
        monkeypatch.setattr(module, "raw_stream", lambda d: (launches.append(now[-1]), raw_stream(d))[1])
    return launches


def test_new_operators_enter_their_tensors_device(elsewhere):
    x = torch.randn(40, 2, 128, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    slots = torch.arange(40, device="cuda")
    cache = fa.Int4KVCache(3, 2, 16, 128)
    out = fa.prompt_attention(x, x, x, cu)
    fa.append_kv_int4(x, x, cache, slots)
    k, v = fa.read_kv_int4(cache, slots)
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    got, lse = fa.paged_attention_int4(x[-1:], cache, cu[1:], table, return_lse=True)
    assert elsewhere == [0] * 4
    assert torch.equal(k, v) and (k - x).abs().max() < 0.5
    assert out.shape == (40, 2, 128) and (got[0] - out[-1]).abs().max() < 1 and lse.isfinite().all()


def test_older_operators_enter_their_tensors_device(elsewhere, monkeypatch):
    monkeypatch.setattr(_torch, "current_device", lambda: elsewhere.now[-1], raising=False)
    stream_of = _torch.stream_of
    for module in (paged, split_kv, mla):
        monkeypatch.setattr(module, "stream_of",
                            lambda t: (elsewhere.append(elsewhere.now[-1]), stream_of(t))[1])
    r = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)  # noqa: E731
    table = torch.arange(2, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    pool = r(2, 2, 16, 128)
    fa.paged_attention(r(1, 4, 128), pool, r(2, 2, 16, 128), lens, table, 0.1, 20)
    fa.paged_attention(query=r(1, 4, 128), key_cache=pool, value_cache=r(2, 2, 16, 128),
                       context_lens=lens, block_tables=table, attn_scale=0.1, max_context_len=20)
    fa.flash_attention(r(1, 4, 1, 128), r(1, 2, 50, 128), r(1, 2, 50, 128))
    latent = r(2, 64, 1, 576)
    fa.append_kv_rows(r(3, 576), latent, torch.arange(3, device="cuda"))
    meta, splits = fa.get_mla_metadata(lens, 16, 1)
    fa.flash_mla_with_kvcache(r(1, 1, 16, 576), latent, table, lens, 512, meta, splits)
    torch.cuda.synchronize()
    assert elsewhere and not any(elsewhere)
