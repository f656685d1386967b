"""Calls made while another device is current launch on their tensors' device.

One GPU is enough: the current device is a number that the tests keep, and
entering a device changes only that number, so nothing runs anywhere else.
"""

import pytest
import torch

import flagattention_b200 as fa
from flagattention_b200 import _torch, kv4, prompt

pytestmark = pytest.mark.gpu


@pytest.fixture
def elsewhere(monkeypatch):
    """Device 1 is current; returns the devices that were current at each launch."""
    now, launches = [1], []

    class Entered:
        def __init__(self, device):
            self.device = torch.device("cuda", device).index if isinstance(device, int) else device.index

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
