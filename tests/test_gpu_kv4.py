"""The 4-bit cache: writes and reads bit for bit, the decode against 64 bits.

Quantisation is defined in f32 with IEEE division, so append + read is compared
for equality with the same formula in torch.  The attention's bound is derived:
with p the softmax weights, c / lo / s the codes, minima and scales, u the unit
roundoff of the output type (2^-8 bf16, 2^-11 f16):
  * p * s is rounded to f16 before the value product (f16 caches: to two f16
    parts, at least 2^-16): u_p * sum p s c, u_p = 2^-11 or 2^-16;
  * the output is rounded: u |o|;
  * f32 accumulation: 2^-20 sum p (|lo| + 47 s);
  * scores are off by at most e = 2^-21 (3 S + 2), S = scale * sum_d |q_d| (47 s
    + |lo|): a weight by 2 e.
"""

import numpy as np
import pytest
import torch

import flagattention_b200 as fa
from flagattention_b200._torch import read_status

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
UP = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -16}
SHAPES = [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32), (256, 128), (256, 64)]


def quantise(x, group):
    """(codes, lo, scale) in f32, groups of the last dim."""
    y = x.float().unflatten(-1, (-1, group))
    lo, hi = y.amin(-1), y.amax(-1)
    scale = ((hi - lo) / 15).to(x.dtype).float()
    c = ((y - lo[..., None]) / scale[..., None]).round().clamp(0, 15)
    return torch.where(scale[..., None] == 0, torch.zeros_like(c), c), lo, scale


def values(x, group):
    c, lo, scale = quantise(x, group)
    return (lo[..., None] + c * scale[..., None]).flatten(-2)


def rows(n, heads, d, dtype, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn(n, heads, d, generator=g, device="cuda") + \
        2 * torch.randn(heads, d, generator=g, device="cuda")
    v = torch.randn(n, heads, d, generator=g, device="cuda") * size
    return k.to(dtype), v.to(dtype)


def same(a, b):
    return torch.equal(a.nan_to_num(12345.0), b.nan_to_num(12345.0)) and \
        torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d, group", SHAPES)
@pytest.mark.parametrize("heads, block, n", [(1, 16, 1), (3, 48, 200), (8, 64, 1000)])
def test_append_then_read_is_exact(d, group, heads, block, n, dtype):
    blocks = -(-n // block) + 2
    cache = fa.Int4KVCache(blocks, heads, block, d, dtype=dtype, group_size=group)
    k, v = rows(n, heads, d, dtype, 1)
    slots = torch.randperm(blocks * block, device="cuda")[:n]
    assert fa.append_kv_int4(k, v, cache, slots) is cache
    for got, x in zip(fa.read_kv_int4(cache, slots), (k, v)):
        assert same(got, values(x, group).to(dtype))
    # the other slots were not touched
    rest = torch.ones(blocks * block, dtype=torch.bool, device="cuda")
    rest[slots] = False
    for got in fa.read_kv_int4(cache, rest.nonzero()[:, 0]):
        assert not got.any()


@pytest.mark.parametrize("d, group", SHAPES)
def test_tile_layout(d, group):
    """The bytes of a tile are where csrc/kv4.cuh says: key words, value units,
    (lo, scale) pairs."""
    cache = fa.Int4KVCache(1, 1, 16, d, group_size=group)
    k, v = rows(16, 1, d, torch.bfloat16, 3)
    fa.append_kv_int4(k, v, cache, torch.arange(16, device="cuda"))
    tile = cache.data[0, 0, 0].cpu().numpy()
    (ck, lk, sk), (cv, lv, sv) = ([t[:, 0].cpu() for t in quantise(x, group)] for x in (k, v))
    ck, cv = (c.flatten(-2).numpy().astype(np.uint8) for c in (ck, cv))
    want = np.zeros_like(tile)
    plane, half_bytes = min(d, 128), 8 * d
    for t in range(16):
        for dim in range(0, d, 2):                        # two codes a byte
            j = dim // 8                                   # key word: dims 8 j .. 8 j + 7
            pl, jj = j // (plane // 8), j % (plane // 8)
            at = pl * 8 * plane + t * (plane // 2) + ((jj % 4) * (plane // 32) + jj // 4) * 4
            want[at + dim % 8 // 2] = ck[t, dim] | ck[t, dim + 1] << 4
            # value dim 64 u + 32 p + 4 r + 2 half + (n & 1), n = 2 p + (n & 1)
            u, p, r, half = dim // 64, dim // 32 % 2, dim % 32 // 4, dim % 4 // 2
            idx = ((t // 8) * (d // 64) + u) * 2 + half
            at = idx // 4 * 512 + (r * 4 + t % 8 // 2) * 16 + idx % 4 * 4 + t % 2 * 2
            want[half_bytes + at + p] = cv[t, dim] | cv[t, dim + 1] << 4
        pairs = torch.stack([torch.cat([lk[t], lv[t]]), torch.cat([sk[t], sv[t]])], -1)
        n = pairs.numel() * 2
        want[2 * half_bytes + t * n:2 * half_bytes + (t + 1) * n] = \
            pairs.to(torch.bfloat16).view(torch.uint8).numpy().ravel()
    assert np.array_equal(tile, want)


def test_skipped_slots_overwrites_and_strides():
    cache = fa.Int4KVCache(4, 2, 32, 128)
    qkv = torch.randn(50, 8, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    qkv = qkv.to(torch.bfloat16)
    k, v = qkv[:, 4:6], qkv[:, 6:]                       # views of a fused projection
    slots = torch.arange(50, device="cuda") + 7
    slots[[3, 20]] = torch.tensor([-1, 4 * 32], device="cuda")   # padding; past the pool
    fa.append_kv_int4(k, v, cache, slots)
    gk, gv = fa.read_kv_int4(cache, slots)
    wk, wv = values(k, 64).to(k.dtype), values(v, 64).to(v.dtype)
    for w in (wk, wv):
        w[[3, 20]] = 0
    assert same(gk, wk) and same(gv, wv)
    fa.append_kv_int4(v, k, cache, slots)                # every bit of a row is replaced
    gk, gv = fa.read_kv_int4(cache, slots)
    assert same(gk, wv) and same(gv, wk)
    odd = torch.randn(51 * 2 * 128 + 1, device="cuda").to(torch.bfloat16)[1:]
    x = odd[:50 * 256].view(50, 2, 128)                  # off 16-byte alignment
    fa.append_kv_int4(x, x, cache, slots)
    assert same(fa.read_kv_int4(cache, slots)[0][:3], values(x, 64).to(x.dtype)[:3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_constant_extreme_and_non_finite_groups(dtype):
    cache = fa.Int4KVCache(1, 1, 16, 128, dtype=dtype)
    top = torch.finfo(dtype).max
    x = torch.randn(8, 1, 128, device="cuda").to(dtype)
    x[0] = 3.25                                          # one value: scale 0, exact
    x[1] = 0
    x[2, 0, ::2], x[2, 0, 1::2] = top, -top              # max - min passes the type's range
    x[3, 0, 5] = float("nan")
    x[4, 0, 70] = float("inf")
    x[5, 0, 7] = -float("inf")
    x[6] = torch.finfo(dtype).tiny                       # smallest normal
    x[7, 0, ::2], x[7, 0, 1::2] = 100, 101               # narrow range far from 0
    slots = torch.arange(8, device="cuda")
    fa.append_kv_int4(x, x, cache, slots)
    for got in fa.read_kv_int4(cache, slots):
        assert same(got[0], x[0]) and same(got[1], x[1]) and same(got[6], x[6])
        # 15 * scale reaches the top within the rounding of the scale
        err = (got[2].float() / top - x[2].float() / top).abs().max()
        assert got[2].isfinite().all() and err <= 2.0 ** -6
        assert got[3, 0, :64].isnan().all() and got[3, 0, 64:].isfinite().all()
        assert got[4, 0, 64:].isnan().all() and got[4, 0, :64].isfinite().all()
        assert got[5, 0, :64].isnan().all() and got[5, 0, 64:].isfinite().all()
        assert (got[7].float() - x[7].float()).abs().max() <= 1 / 30 + 0.5 * (dtype == torch.bfloat16)


def test_subnormal_ranges():
    """Groups whose range is a few subnormal steps: the scale rounds to one too."""
    cache = fa.Int4KVCache(1, 1, 16, 64)
    steps = torch.arange(64, device="cuda") % torch.tensor([2, 7, 16, 40], device="cuda")[:, None]
    x = (steps * 2.0 ** -133).to(torch.bfloat16)[:, None]  # bf16's smallest numbers
    assert x.float().max() > 0
    fa.append_kv_int4(x, x, cache, torch.arange(4, device="cuda"))
    for got in fa.read_kv_int4(cache, torch.arange(4, device="cuda")):
        assert same(got, values(x, 64).to(x.dtype))


@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_scale(dtype, signed):
    """Codes are those of IEEE division for every scale that the type has: a group for
    each of its positive numbers as the largest value, beside random ones down to 0
    or to its negative."""
    bits = torch.arange(1, 0x7f80 if dtype is torch.bfloat16 else 0x7c00, device="cuda")
    top = bits.to(torch.int16).view(dtype)
    if signed:
        top = top[top.double() <= torch.finfo(dtype).max / 2]
    n = top.shape[0]
    g = torch.Generator(device="cuda").manual_seed(21)
    part = torch.rand(n, 64, generator=g, device="cuda", dtype=torch.float64)
    x = (part * 2 - 1 if signed else part) * top.double()[:, None]
    x[:, 17], x[:, 40] = top.double(), -top.double() if signed else 0.0
    x = x.to(dtype)[:, None]
    cache = fa.Int4KVCache(-(-n // 16), 1, 16, 64, dtype=dtype)
    slots = torch.arange(n, device="cuda")
    fa.append_kv_int4(x, x.flip(-1), cache, slots)
    for got, rows_ in zip(fa.read_kv_int4(cache, slots), (x, x.flip(-1))):
        want = values(rows_, 64).to(dtype)
        assert torch.equal(got, want.clamp(max=torch.finfo(dtype).max))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_subnormal_scales(dtype):
    """Ranges of 1 .. 255 of the type's smallest steps: a scale of a few steps is
    off by up to half a step (22 steps: 1.47 rounds to 1), so the largest quotient
    passes 15 by up to half again and is cut there."""
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    tops = torch.arange(1, 256, device="cuda")[:, None]
    dim = torch.arange(64, device="cuda")
    n = torch.where(dim % 9 == 4, tops, dim * dim % (tops + 1))   # the largest beside others
    x = (n.double() * step).to(dtype)[:, None]
    assert torch.equal(x.double()[:, 0], n.double() * step)
    cache = fa.Int4KVCache(16, 1, 16, 64, dtype=dtype)
    slots = torch.arange(255, device="cuda")
    fa.append_kv_int4(x, -x, cache, slots)
    for got, rows_ in zip(fa.read_kv_int4(cache, slots), (x, -x)):
        assert same(got, values(rows_, 64).to(dtype))


def build(lens, hq, hk, d, group, block, dtype, seed=0, size=1.0, pool_extra=3):
    """Cache with shuffled pages whose unused slots hold NaN scales and any
    codes, the query, and the rows of each sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = [-(-n // block) for n in lens]
    blocks = sum(per) + pool_extra
    cache = fa.Int4KVCache(blocks, hk, block, d, dtype=dtype, group_size=group)
    cache.data.fill_(0xff)                               # bf16 / f16 0xffff is a NaN
    perm = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(per + [1]), dtype=torch.int32, device="cuda")
    data, a = [], 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = perm[a:a + per[b]]
        a += per[b]
        k, v = rows(n, hk, d, dtype, seed * 1000 + b, size)
        t = torch.arange(n, device="cuda")
        fa.append_kv_int4(k, v, cache, table[b].long()[t // block] * block + t % block)
        data.append((k, v))
    q = torch.randn(len(lens), hq, d, generator=g, device="cuda").to(dtype)
    return cache, table, q, data, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(cache, table, q, data, lens, scale=None, live=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = fa.paged_attention_int4(q, cache, lens, table, scale, return_lse=True)
    torch.cuda.synchronize()
    assert read_status(torch.device("cuda")) == 0
    hq, hk, group = q.shape[1], cache.num_kv_heads, cache.group_size
    for b, (k, v) in enumerate(data):
        if live is not None:                              # tokens that count
            k, v = k[live[b]], v[live[b]]
        if k.shape[0] == 0:
            assert not out[b].any() and (lse[b] == -np.inf).all()
            continue
        (ck, lk, sk), (cv, lv, sv) = ([t.double() for t in quantise(x, group)] for x in (k, v))
        wide = lambda t: t[..., None].expand(*t.shape, group).flatten(-2)  # noqa: E731
        heads = lambda t: t.transpose(0, 1).repeat_interleave(hq // hk, 0)  # noqa: E731
        ck, cv = ck.flatten(-2), cv.flatten(-2)
        kk, vv = (heads(wide(lo) + c * wide(s)) for c, lo, s in ((ck, lk, sk), (cv, lv, sv)))
        q64 = q[b].double()[:, None]                      # [hq, 1, d]
        s = scale * q64 @ kk.transpose(1, 2)              # [hq, 1, n]
        p, want_l = torch.softmax(s, -1), torch.logsumexp(s, -1)
        want = (p @ vv)[:, 0]
        size = scale * q64.abs() @ heads(47 * wide(sk) + wide(lk).abs()).transpose(1, 2)
        err = 2.0 ** -21 * (3 * size.amax(-1, keepdim=True) + 2)
        mag = (p @ heads(wide(lv).abs() + 47 * wide(sv)))[:, 0]
        tol = 1.01 * (UP[q.dtype] * (p @ heads(cv * wide(sv)))[:, 0] + U[q.dtype] * want.abs()) + \
            (2 * err[:, 0] + 2.0 ** -20) * mag + 1e-7
        off = (out[b].double() - want).abs()
        assert (off <= tol).all(), f"sequence {b}: {(off / tol).max():.2f} of the bound"
        off_l = (lse[b].double() - want_l[:, 0]).abs()
        assert (off_l <= err[:, 0, 0] + 2.0 ** -21 * want_l[:, 0].abs()).all(), off_l.max()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d, group", SHAPES)
@pytest.mark.parametrize("hq, hk", [(8, 1), (3, 3), (40, 2)])
def test_decode_shapes(d, group, hq, hk, dtype):
    lens = [1, 15, 16, 17, 63, 64, 65, 0, 200, 513]
    check(*build(lens, hq, hk, d, group, 16, dtype, seed=1))


@pytest.mark.parametrize("group_heads", [1, 2, 7, 8, 9, 16, 17, 64])
def test_decode_group_sizes(group_heads):
    check(*build([5, 300, 77], 2 * group_heads, 2, 128, 64, 32, torch.bfloat16, seed=2))


@pytest.mark.parametrize("block", [16, 32, 48, 64, 256])
def test_decode_pages(block):
    check(*build([1, 31, 255, 700, 1500], 16, 2, 128, 64, block, torch.bfloat16, seed=3))


@pytest.mark.parametrize("lens", [[20000], [9000, 1, 0, 12000], [0, 0, 0], [0, 5, 0, 0],
                                  [1 + (i * 53) % 300 for i in range(400)]])
def test_decode_long_split_and_many(lens):
    check(*build(lens, 8, 2, 64, 32, 16, torch.bfloat16, seed=4))


@pytest.mark.parametrize("d, group", [(128, 64), (64, 32), (256, 128)])
@pytest.mark.parametrize("dtype, bound", [(torch.bfloat16, 3e-3), (torch.float16, 1e-3)])
def test_decode_long_context_keeps_its_accuracy(d, group, dtype, bound):
    """Over many tokens the output is the small difference of large sums (codes
    and minima are not centred): 2-norm against 64 bits, one sequence spread over
    the GPU and a batch of which every CTA holds whole ones (one sequence's sums
    run over hundreds of tiles in one warp).  Expected: the output's
    rounding (at most 2^-8 or 2^-11, 2^-8 / sqrt(3) = 2.3e-3 or 2.8e-4 over the
    mantissas), P' rounded to 16 bits (independent: 2^-11 / sqrt(3) * rms(s c) /
    rms(v) = 7e-4, or nothing), and f32 sums of n / 64 products per warp, each off
    by 2^-24 of a sum about 2 / rms(o) = 60 times the output: below 5e-4.  Sums that a
    warp lets grow further have to be split."""
    cache, table, q, data, lens = build([40000], 8, 1, d, group, 64, dtype, seed=12)
    k, v = (_exact(x[:, 0], group) for x in data[0])
    p = torch.softmax(q[0].double() @ k.T * d ** -0.5, -1)
    want = p @ v
    for batch in (1, 1500):                               # the same pages for all
        out = fa.paged_attention_int4(q.expand(batch, -1, -1), cache, lens.expand(batch),
                                      table.expand(batch, -1))
        for b in {0, batch // 2, batch - 1}:
            assert (out[b].double() - want).norm() / want.norm() <= bound


def _exact(x, group):
    c, lo, s = (t.double() for t in quantise(x, group))
    return (lo[..., None] + c * s[..., None]).flatten(-2)


@pytest.mark.parametrize("lens", [[4001], [900] * 9, [33, 5000, 0, 1]])
@pytest.mark.parametrize("d, group, hq", [(64, 32, 4), (64, 64, 40), (128, 128, 4), (256, 64, 6)])
def test_decode_merges_of_many_and_few_pieces(d, group, hq, lens):
    check(*build(lens, hq, 2, d, group, 16, torch.bfloat16, seed=18))


def test_decode_sharp_scores():
    """Scores spread over hundreds, rising and falling along the context."""
    cache, table, q, data, lens = build([900, 640], 8, 2, 128, 64, 16, torch.bfloat16, seed=5)
    check(cache, table, q * 30, data, lens)
    for b, (k, v) in enumerate(data):
        n = k.shape[0]
        ramp = torch.linspace(8, 0.1, n, device="cuda")[:, None, None]
        data[b] = ((k * ramp).to(k.dtype), v)
        t = torch.arange(n, device="cuda")
        fa.append_kv_int4(*data[b], cache, table[b].long()[t // 16] * 16 + t % 16)
    check(cache, table, q * 4, data, lens)


@pytest.mark.parametrize("size", [1e-4, 1e4])
def test_decode_f16_range(size):
    """Value scales far below and above 1 in f16 (products p * s leave f16's
    accurate range)."""
    check(*build([400, 33], 8, 1, 128, 64, 16, torch.float16, seed=6, size=size))


@pytest.mark.parametrize("dtype, factor, bound", [(torch.bfloat16, 1e3, 3e-3), (torch.bfloat16, 1e5, 3e-3),
                                                  (torch.float16, 1e4, 1e-3)])
@pytest.mark.parametrize("d, group, hq", [(128, 64, 8), (64, 32, 8), (256, 64, 8), (128, 32, 40)])
@pytest.mark.parametrize("kind", ["first token", "middle token", "group", "some heads' token"])
def test_decode_values_of_very_different_sizes(kind, d, group, hq, dtype, factor, bound):
    """Large value rows that nobody or only some heads attend to, or one large
    group, take nothing from the rest.  2-norm against 64 bits of every head and
    group by itself; the bound is that of
    ``test_decode_long_context_keeps_its_accuracy``: what is added, products p * s
    that are small next to the largest one of their head and group, is off by
    15 * 2^-28 of that per token, 2^-28 * 15 sqrt(20000) = 8e-6 together.  One
    sequence spread over the GPU, and a batch of which every CTA holds whole ones."""
    n, hk = 20000, 2
    cache, table, q, data, lens = build([n], hq, hk, d, group, 64, dtype, seed=19)
    (k, v), = data
    q *= 3                                                # scores of standard deviation 3
    q[..., 0] = 8
    if kind == "some heads' token":
        q[:, 1::2, 0] = -8                                # the even heads see only that token
    far = 40 * d ** 0.5 / 8                               # scores 40 apart
    k[..., 0] = 0
    if kind == "group":
        v[..., :group] *= factor
    else:
        t = 0 if kind == "first token" else n // 2
        k[t, :, 0] = far if kind == "some heads' token" else -far
        v[t, :, :group if kind == "some heads' token" else d] *= factor
    t = torch.arange(n, device="cuda")
    fa.append_kv_int4(k, v, cache, table[0].long()[t // 64] * 64 + t % 64)
    kk, vv = (_exact(x, group).transpose(0, 1).repeat_interleave(hq // hk, 0) for x in (k, v))
    p = torch.softmax(d ** -0.5 * q[0].double()[:, None] @ kk.transpose(1, 2), -1)
    want = (p @ vv)[:, 0].unflatten(-1, (-1, group))
    for batch in (1, 600):                                # the same pages for all
        out = fa.paged_attention_int4(q.expand(batch, -1, -1), cache, lens.expand(batch),
                                      table.expand(batch, -1))
        for b in {0, batch // 2, batch - 1}:
            off = (out[b].double().unflatten(-1, (-1, group)) - want).norm(dim=-1) / want.norm(dim=-1)
            assert (off <= bound).all(), off.max()


@pytest.mark.parametrize("dtype, bound", [(torch.bfloat16, 2.0 ** -20), (torch.float16, 2.0 ** -22)])
@pytest.mark.parametrize("d, group, hq", [(64, 32, 16), (64, 64, 64), (128, 128, 32), (256, 64, 8)])
def test_log_sum_exp_of_short_contexts(d, group, hq, dtype, bound):
    """2-norm of the log-sum-exp's error against 64 bits.  A score is the small
    difference of two sums about ten times as large, each in f32 over d products
    (simulated with exact products, one rounding per 16 dims: 1e-7 of the scores) and the
    logarithm adds 2^-22 of a binary unit at most: 2^-22 in all.  bf16 caches, whose codes'
    products lose bits 24 below the largest operands' exponents: four times that."""
    lens = [1 + b % 13 for b in range(60)]
    cache, table, q, data, n = build(lens, hq, 4, d, group, 16, dtype, seed=23)
    _, lse = fa.paged_attention_int4(q, cache, n, table, return_lse=True)
    want = torch.empty_like(lse, dtype=torch.float64)
    for b, (k, _) in enumerate(data):
        kk = _exact(k, group).transpose(0, 1).repeat_interleave(hq // 4, 0)
        want[b] = torch.logsumexp(d ** -0.5 * q[b].double()[:, None] @ kk.transpose(1, 2), -1)[:, 0]
    assert (lse.double() - want).norm() / want.norm() <= bound


@pytest.mark.parametrize("size", [1e-30, 1e33])
@pytest.mark.parametrize("lens", [[3000], [3000] * 300])
def test_decode_bf16_range(size, lens):
    """Value rows near both ends of bf16's range; the bound of
    ``test_decode_long_context_keeps_its_accuracy``, which is relative."""
    cache, table, q, data, n = build([3000], 8, 1, 128, 64, 16, torch.bfloat16, seed=22, size=size)
    k, v = (_exact(x[:, 0], 64) for x in data[0])
    want = torch.softmax(q[0].double() @ k.T * 128 ** -0.5, -1) @ v
    batch = len(lens)
    out = fa.paged_attention_int4(q.expand(batch, -1, -1), cache, n.expand(batch),
                                  table.expand(batch, -1))
    for b in {0, batch - 1}:
        assert ((out[b].double() - want) / size).norm() / (want / size).norm() <= 3e-3


def test_decode_nan_stays_and_does_not_spread():
    lens = [50, 70]
    cache, table, q, data, n = build(lens, 4, 2, 128, 64, 16, torch.bfloat16, seed=7)
    k = data[0][0].clone()
    k[20, 0, 3] = float("nan")
    fa.append_kv_int4(k[20:21], data[0][1][20:21], cache,
                      (table[0, 1].long() * 16 + 4).reshape(1))
    out, lse = fa.paged_attention_int4(q, cache, n, table, return_lse=True)
    assert out[0, :2].isnan().all() and lse[0, :2].isnan().all()     # kv head 0
    assert out[0, 2:].isfinite().all() and out[1].isfinite().all() and lse[1].isfinite().all()


@pytest.mark.parametrize("lens", [[9000], [2500] * 12])    # wide and narrow merges
def test_decode_nan_stays_when_entries_are_split(lens):
    cache, table, q, data, n = build(lens, 16, 2, 128, 64, 16, torch.bfloat16, seed=17)
    k = data[0][0].clone()
    k[20, 0, 3] = float("nan")                                       # in one piece of kv head 0
    fa.append_kv_int4(k[20:21], data[0][1][20:21], cache,
                      (table[0, 1].long() * 16 + 4).reshape(1))
    q[0, 9] = float("nan")                                           # in every piece of its row
    out, lse = fa.paged_attention_int4(q, cache, n, table, return_lse=True)
    bad = torch.zeros(len(lens), 16, dtype=torch.bool, device="cuda")
    bad[0, :8] = bad[0, 9] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(lse.isnan(), bad) and lse[~bad].isfinite().all()


def test_decode_table_entries_outside_the_pool_and_short_tables():
    cache, table, q, data, lens = build([100, 64, 40], 4, 2, 64, 32, 16, torch.bfloat16, seed=8)
    live = [torch.ones(n, dtype=torch.bool, device="cuda") for n in (100, 64, 40)]
    table[0, 2], table[1, 0] = -1, cache.num_blocks
    live[0][32:48] = False
    live[1][:16] = False
    check(cache, table, q, data, lens, live=live)
    lens[0] = 1000                                        # more tokens than the table names
    live[0][:] = True
    table, lens = table[:1, :2].contiguous(), lens[:1]
    check(cache, table, q[:1], [(data[0][0][:32], data[0][1][:32])], lens)
    lens[0] = -5
    check(cache, table, q[:1], [(data[0][0][:0], data[0][1][:0])], lens)


def test_decode_views_streams_and_graph():
    cache, table, q, data, lens = build([300, 45], 8, 2, 128, 64, 16, torch.bfloat16, seed=9)
    first = check(cache, table, q, data, lens)
    fused = torch.zeros(2, 12, 128, dtype=q.dtype, device="cuda")
    fused[:, 2:10] = q
    wide = torch.zeros(2, 50, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    assert torch.equal(first, fa.paged_attention_int4(fused[:, 2:10], cache, lens,
                                                      wide[:, :table.shape[1]]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = fa.paged_attention_int4(q, cache, lens, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = fa.paged_attention_int4(q, cache, lens, table)
    lens.copy_(torch.tensor([17, 45], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, fa.paged_attention_int4(q, cache, lens, table))


def test_pool_past_32_bit_offsets():
    """Blocks beyond 4 GiB of the pool."""
    block, hk, d = 256, 8, 128
    per = hk * block * 144
    blocks = (5 << 30) // per
    cache = fa.Int4KVCache(blocks, hk, block, d)
    k, v = rows(300, hk, d, torch.bfloat16, 10)
    table = torch.tensor([[blocks - 1, blocks - 7]], dtype=torch.int32, device="cuda")
    t = torch.arange(300, device="cuda")
    slots = table[0].long()[t // block] * block + t % block
    fa.append_kv_int4(k, v, cache, slots)
    assert same(fa.read_kv_int4(cache, slots)[0], values(k, 64).to(k.dtype))
    q = torch.randn(1, 64, d, device="cuda").to(torch.bfloat16)
    check(cache, table, q, [(k, v)], torch.tensor([300], dtype=torch.int32, device="cuda"))


def test_refusals():
    for bad in (dict(block_size=24), dict(head_size=96), dict(group_size=16),
                dict(head_size=64, group_size=128), dict(head_size=256, group_size=32),
                dict(dtype=torch.float32)):
        args = dict(num_blocks=2, num_kv_heads=2, block_size=16, head_size=128, group_size=64)
        args.update(bad)
        with pytest.raises(fa.Unsupported):
            fa.Int4KVCache(**args)
    with pytest.raises(fa.InvalidArgument):
        fa.Int4KVCache(2, 0, 16, 128)
    with pytest.raises(fa.InvalidArgument):
        fa.Int4KVCache(2, 2, 16, 128, device="cpu")
    cache = fa.Int4KVCache(2, 2, 16, 128)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    for k, v, s in ((x.half(), x, slots), (x, x[:, :1], slots), (x, x, slots.int()),
                    (x[:2], x, slots), (x, x, slots.cpu())):
        with pytest.raises(fa.InvalidArgument):
            fa.append_kv_int4(k, v, cache, s)
    with pytest.raises(fa.InvalidArgument):
        fa.read_kv_int4(cache, slots.int())
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for args in ((q[:, :3], lens, table), (q.half(), lens, table), (q[..., :64], lens, table),
                 (q, lens.long(), table), (q, lens, table.long()), (q, lens[:0], table),
                 (q, lens, table[0])):
        with pytest.raises(fa.InvalidArgument):
            fa.paged_attention_int4(args[0], cache, args[1], args[2])
    with pytest.raises(fa.InvalidArgument):
        fa.paged_attention_int4(q, cache, lens, table, attn_scale=0.0)
    fa.append_kv_int4(x[:0], x[:0], cache, slots[:0])
    assert fa.read_kv_int4(cache, slots[:0])[0].shape == (0, 2, 128)
    assert fa.paged_attention_int4(q[:0], cache, lens[:0], table[:0]).shape == (0, 4, 128)
