"""Prompts of different lengths, then decode steps, over a 4-bit cache.

One attention layer with random weights: a step's prompts are packed and
attended with ``prompt_attention``, their key / value rows go to an
``Int4KVCache``, and each decode step appends one token per sequence and attends
with ``paged_attention_int4``.  A later chunk of a prompt reads its cached context
back with ``read_kv_int4``.  The same steps over 16-bit pages (``paged_attention``)
show what the 4 bits change.

    python examples/prompt_then_int4_decode.py [--steps 8]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import flagattention_b200 as fa  # noqa: E402


class Layer:
    """Projections of one attention layer (grouped-query heads)."""

    def __init__(self, width, heads, kv_heads, head, dtype, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head = heads, kv_heads, head
        self.w = (torch.randn(width, (heads + 2 * kv_heads) * head, generator=g, device="cuda") /
                  width ** 0.5).to(dtype)

    def qkv(self, x):
        """q, k, v as views of one fused projection."""
        rows = (x @ self.w).view(x.shape[0], -1, self.head)
        return rows.split([self.heads, self.kv_heads, self.kv_heads], dim=1)


def slots_of(table, block, sequence, first, count):
    """Pool slots of tokens first .. first + count - 1 of a sequence."""
    t = torch.arange(first, first + count, device="cuda")
    return table[sequence].long()[t // block] * block + t % block


def run(lens=(37, 500, 129), steps=8, width=512, heads=16, kv_heads=2, head=128, block=16,
        dtype=torch.bfloat16):
    """Returns (4-bit, 16-bit) outputs of the last decode step and of a second
    prompt chunk over the cached context, and the cache sizes in bytes."""
    g = torch.Generator(device="cuda").manual_seed(1)
    layer = Layer(width, heads, kv_heads, head, dtype)
    batch, chunk = len(lens), 20
    per = -(-(max(lens) + steps + chunk) // block)
    table = torch.randperm(batch * per, generator=g, device="cuda").to(torch.int32).view(batch, per)
    cache = fa.Int4KVCache(batch * per, kv_heads, block, head, dtype=dtype)
    k16 = torch.zeros(batch * per, kv_heads, block, head, dtype=dtype, device="cuda")
    v16 = torch.zeros_like(k16)

    def store(k, v, slots):
        fa.append_kv_int4(k, v, cache, slots)
        k16[slots // block, :, slots % block] = k
        v16[slots // block, :, slots % block] = v

    # the prompts, packed
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(lens), width, generator=g, device="cuda").to(dtype)
    q, k, v = layer.qkv(x)
    fa.prompt_attention(q, k, v, cu)
    store(k, v, torch.cat([slots_of(table, block, b, 0, n) for b, n in enumerate(lens)]))

    # decode steps: one token per sequence
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        x = torch.randn(batch, width, generator=g, device="cuda").to(dtype)
        q, k, v = layer.qkv(x)
        at = seq.long()
        store(k, v, table.long().gather(1, (at // block)[:, None])[:, 0] * block + at % block)
        seq += 1
        out4 = fa.paged_attention_int4(q, cache, seq, table)
        out16 = fa.paged_attention(q, k16, v16, seq, table, head ** -0.5, int(max(lens) + steps))

    # the next chunk of sequence 0: its context comes back from the cache
    n = lens[0] + steps
    x = torch.randn(chunk, width, generator=g, device="cuda").to(dtype)
    q, k, v = layer.qkv(x)
    slots = slots_of(table, block, 0, n, chunk)
    store(k, v, slots)
    all_slots = slots_of(table, block, 0, 0, n + chunk)
    offsets = torch.tensor([0, chunk], dtype=torch.int32, device="cuda")
    keys = torch.tensor([0, n + chunk], dtype=torch.int32, device="cuda")
    chunk4 = fa.prompt_attention(q, *fa.read_kv_int4(cache, all_slots), offsets, keys)
    chunk16 = fa.prompt_attention(q, k16[all_slots // block, :, all_slots % block],
                                  v16[all_slots // block, :, all_slots % block], offsets, keys)
    return (out4, out16), (chunk4, chunk16), (cache.data.numel(), 4 * k16.numel())


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--steps", type=int, default=8)
    decode, chunk, size = run(steps=p.parse_args().steps)
    for name, (a, b) in (("last decode step", decode), ("second prompt chunk", chunk)):
        d = (a.float() - b.float()).norm() / b.float().norm()
        print(f"{name}: 4-bit against 16-bit cache, relative difference {d:.3f}")
    print(f"cache: {size[0]} bytes in 4 bits, {size[1]} in 16")


if __name__ == "__main__":
    main()
