"""prompt_attention (csrc/prompt.cu) against the definition in 64 bits.

Lengths 0, 1 and around the tile edges, more queries than keys (rows that see
nothing), earlier keys (a later chunk of a prompt), group sizes that do and do
not divide a tile, padded head sizes, strided and misaligned views, values
that must not leak from one packed sequence into the next.

The bound is elementwise and derived, not tuned.  With u the unit roundoff of
the output type (8 significant bits in bf16: 2^-8; 11 in f16: 2^-11), p the
softmax weights and a = sum_j p_j |v_j|:
  * probabilities are rounded to the input type before the value product,
    while their sum is not: u * a;
  * f16 probabilities under 2^-14 are rounded to multiples of 2^-24 instead;
    the row sum is at least 1 in their units: 2^-25 n max|v|  (f16);
  * the output is rounded: u * |o|;
  * f32 scores: each is off by at most e = 2^-21 * scale * sum_d |q_d k_d|
    (accumulation over at most 192 products) + 2^-21 * (its own size in log2
    units, and the approximate exponential): a weight by 2 e, so 2 e a.
"""

import numpy as np
import pytest
import torch

import flagattention_b200 as fa
from flagattention_b200._torch import read_status

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(q, k, v, lens_q, lens_k, causal, scale):
    """(o, lse, bound of |o|'s error, bound of lse's error) in f64, packed."""
    f16 = q.dtype == torch.float16
    q, k, v = q.double(), k.double(), v.double()
    (total, hq, _), hk, dv = q.shape, k.shape[1], v.shape[2]
    group = hq // hk
    o = torch.zeros(total, hq, dv, dtype=torch.float64, device=q.device)
    lse = torch.full((hq, total), -np.inf, dtype=torch.float64, device=q.device)
    tol_p, tol_a = torch.zeros_like(o), torch.zeros_like(o)
    tol_l = torch.zeros_like(lse)
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        if n and m:
            qs = q[a:a + n].transpose(0, 1)
            ks = k[b:b + m].transpose(0, 1).repeat_interleave(group, 0)
            vs = v[b:b + m].transpose(0, 1).repeat_interleave(group, 0)
            s = scale * qs @ ks.transpose(1, 2)
            if causal:
                mask = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
                s = s.masked_fill(mask, -np.inf)
            top = s.amax(-1, keepdim=True).clamp(min=-1e300)
            e = (s - top).exp()
            z = e.sum(-1, keepdim=True)
            p = torch.where(z > 0, e / z, torch.zeros_like(e))
            size = scale * qs.abs() @ ks.abs().transpose(1, 2)
            err = 2.0 ** -21 * (size.amax(-1, keepdim=True) * 3 + 2)
            av = p @ vs.abs()
            o[a:a + n] = (p @ vs).transpose(0, 1)
            tol_p[a:a + n] = av.transpose(0, 1)
            tol_a[a:a + n] = (2 * err * av + 2.0 ** -25 * m * vs.abs().max() * f16).transpose(0, 1)
            lse[:, a:a + n] = (top + z.log())[..., 0]
            tol_l[:, a:a + n] = err[..., 0] + 2.0 ** -21 * lse[:, a:a + n].abs().nan_to_num(0, 0, 0)
        a, b = a + n, b + m
    return o, lse, tol_p, tol_a, tol_l


def check(q, k, v, lens_q, lens_k, causal=True, scale=None, skip=()):
    cu = lambda x: torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32, device="cuda")  # noqa: E731
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = fa.prompt_attention(q, k, v, cu(lens_q), cu(lens_k), causal=causal, sm_scale=scale,
                                   return_lse=True)
    torch.cuda.synchronize()
    assert read_status(torch.device("cuda")) == 0
    o, want_l, tol_p, tol_a, tol_l = reference(q, k, v, lens_q, lens_k, causal, scale)
    u = U[q.dtype]
    tol = 1.01 * u * (tol_p + o.abs()) + tol_a + 1e-7
    live = torch.ones(out.shape[0], dtype=torch.bool, device="cuda")
    a = 0
    for i, n in enumerate(lens_q):
        live[a:a + n] = i not in skip
        a += n
    live[a:] = False
    bad = ((out.double() - o).abs() > tol)[live]
    assert not bad.any() and out[live].isfinite().all(), \
        f"{int(bad.sum())} outputs off, worst {((out.double() - o).abs() / tol)[live].max():.2f} of the bound"
    empty = want_l == -np.inf
    assert torch.equal(lse[:, live] == -np.inf, empty[:, live])
    d = (lse.double() - want_l).abs()[:, live][~empty[:, live]]
    assert (d <= tol_l[:, live][~empty[:, live]]).all(), d.max()
    return out, lse


def tensors(lens_q, lens_k, hq, hk, d, dv, dtype, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: (size * torch.randn(*s, generator=g, device="cuda")).to(dtype)  # noqa: E731
    return r(sum(lens_q), hq, d), r(sum(lens_k), hk, d), r(sum(lens_k), hk, dv)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, hk, d, dv", [(8, 8, 128, 128), (16, 2, 128, 128), (4, 4, 64, 64),
                                           (6, 2, 192, 128), (10, 2, 96, 96), (5, 1, 40, 24),
                                           (7, 1, 136, 72), (2, 2, 8, 8)])
def test_lengths_around_tile_edges(hq, hk, d, dv, dtype, causal):
    lens = [1, 0, 127, 128, 129, 2, 255, 256, 257, 300, 31]
    check(*tensors(lens, lens, hq, hk, d, dv, dtype), lens, lens, causal)


@pytest.mark.parametrize("hq, hk", [(128, 1), (64, 1), (48, 1), (33, 1), (40, 8), (24, 8), (9, 3)])
def test_group_sizes(hq, hk):
    lens = [5, 1, 140, 67]
    check(*tensors(lens, lens, hq, hk, 64, 64, torch.bfloat16, seed=1), lens, lens)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq, hk, d, dv", [(8, 1, 128, 128), (2, 2, 64, 64), (3, 3, 192, 128)])
def test_keys_and_queries_differ(hq, hk, d, dv, causal):
    lens_q = [1, 16, 200, 1, 300, 130, 0, 7, 5]
    lens_k = [1000, 129, 700, 1, 3, 0, 50, 2048, 4]   # rows that see nothing, no keys, no queries
    check(*tensors(lens_q, lens_k, hq, hk, d, dv, torch.bfloat16, seed=2), lens_q, lens_k, causal)


@pytest.mark.parametrize("d", [64, 128])
def test_sharp_and_large_scores(d):
    """Scores spread over hundreds: the running maximum moves often, and by
    more than the rescale threshold."""
    lens = [700, 513]
    q, k, v = tensors(lens, lens, 8, 2, d, d, torch.bfloat16, seed=3)
    ramp = torch.linspace(0.1, 6, sum(lens), device="cuda")[:, None, None]
    check(q * 6, (k * ramp).to(k.dtype), v, lens, lens)
    check(q * 6, (k * ramp.flip(0)).to(k.dtype), v, lens, lens)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_neighbours_do_not_leak(value):
    """One packed sequence of NaN / infinities next to finite ones, and such
    rows past the last sequence."""
    lens = [70, 130, 3, 129]
    total = sum(lens) + 40
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(total, 4, 128, generator=g, device="cuda").to(torch.bfloat16)
               for _ in range(3))
    for x in (k, v, q):
        x[lens[0]:lens[0] + lens[1]] = value
        x[sum(lens):] = value
    check(q, k, v, lens, lens, causal=False, skip=(1,))
    check(q, k, v, lens, lens, causal=True, skip=(1,))


@pytest.mark.parametrize("hq, hk, d, dv, dtype", [(8, 8, 128, 128, torch.bfloat16),
                                                  (16, 2, 128, 128, torch.float16),
                                                  (64, 1, 64, 64, torch.bfloat16),
                                                  (4, 4, 192, 128, torch.bfloat16),
                                                  (24, 1, 96, 72, torch.bfloat16),
                                                  (3, 3, 64, 64, torch.float16)])
@pytest.mark.parametrize("lens_q, lens_k", [([300, 70, 130], [300, 70, 130]),
                                            ([40, 260, 9], [515, 300, 5]),
                                            ([100], [9000])])
def test_later_tokens_do_not_reach_earlier_rows(lens_q, lens_k, hq, hk, d, dv, dtype):
    """A causal row's output does not depend on any bit of the keys that it does not
    see.  Infinities and NaN in value rows reach exactly the elements that weigh
    them (an infinity, or a NaN where infinities cancel), NaN keys every element of the rows
    that see them; every other element keeps its bits."""
    q, k, v = tensors(lens_q, lens_k, hq, hk, d, dv, dtype, seed=20)
    cu = lambda x: torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32, device="cuda")  # noqa: E731
    args = cu(lens_q), cu(lens_k)
    clean, clean_l = fa.prompt_attention(q, k, v, *args, return_lse=True)
    inf, nan = float("inf"), float("nan")
    plants = [(0, 3, inf), (0, 3, inf), (0, 5, -inf), (1, 5, inf), (2, 7, nan), (5, 0, nan), (1, dv - 1, nan),
              (40, 9, -inf), (3, 9, -inf)]
    want = clean.double().clone()
    bad_v = v.clone()
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        row = torch.arange(n, device="cuda")
        for back, dim, x in plants:                       # `back` tokens before the last
            t = m - 1 - back * max(1, min(n, m) // 45)
            if t < 0:
                continue
            bad_v[b + t, back % hk, dim] = x
            sees = row + m - n >= t
            heads = torch.arange(hq, device="cuda") // (hq // hk) == back % hk
            want[a:a + n, :, dim] += torch.where(sees[:, None] & heads, x, 0.0)
        a, b = a + n, b + m
    got, got_l = fa.prompt_attention(q, k, bad_v, *args, return_lse=True)
    assert torch.equal(got_l, clean_l)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0, 9, -9), want.to(dtype).nan_to_num(0, 9, -9))
    want, want_l, bad_k, bad_v = clean.double(), clean_l.clone(), k.clone(), v.clone()
    a = b = 0
    for n, m in zip(lens_q, lens_k):                      # the last third's keys and values
        t = m - max(min(n, m) // 3, 1)
        bad_k[b + t:b + m], bad_v[b + t:b + m] = nan, nan
        sees = torch.arange(n, device="cuda") + m - n >= t
        want[a:a + n] = torch.where(sees[:, None, None], nan, clean[a:a + n].double())
        want_l[:, a:a + n] = torch.where(sees, nan, clean_l[:, a:a + n])
        a, b = a + n, b + m
    got, got_l = fa.prompt_attention(q, bad_k, bad_v, *args, return_lse=True)
    for x, y in ((got, want.to(dtype)), (got_l, want_l)):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(0, 9, -9), y.nan_to_num(0, 9, -9))


def test_nan_stays_when_keys_are_split():
    """Few queries over many keys: a NaN in one range of the keys, and one in a
    query, which meets it in every range."""
    n, m = 100, 9000
    q, k, v = tensors([n], [m], 16, 2, 128, 128, torch.bfloat16, seed=14)
    k[5000, 0] = float("nan")
    q[7, 9] = float("nan")
    cu = lambda x: torch.tensor([0, x], dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = fa.prompt_attention(q, k, v, cu(n), cu(m), return_lse=True)
    bad = torch.zeros(n, 16, dtype=torch.bool, device="cuda")
    bad[:, :8] = bad[7, 9] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(lse.isnan(), bad.T) and lse.T[~bad].isfinite().all()


def test_values_of_the_lowest_type_value():
    lens = [100, 260]
    q, k, v = tensors(lens, lens, 4, 2, 64, 64, torch.bfloat16, seed=5)
    k[50:60] = torch.finfo(torch.bfloat16).min / 256   # scores near -1e38: weight 0, no NaN
    q = q.abs()
    check(q, k, v, lens, lens)


def test_views_of_a_fused_projection():
    lens = [200, 77, 129]
    g = torch.Generator(device="cuda").manual_seed(6)
    qkv = torch.randn(sum(lens), 12, 128, generator=g, device="cuda").to(torch.bfloat16)
    check(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], lens, lens)
    flat = torch.randn(sum(lens) * 4 * 64 + 1, generator=g, device="cuda").to(torch.float16)
    x = flat[1:].view(sum(lens), 4, 64)               # rows off 16-byte alignment
    check(x, x[:, :2], x[:, 2:], lens, lens)
    t = torch.randn(4, sum(lens), 64, generator=g, device="cuda").to(torch.float16).transpose(0, 1)
    check(t, t, t, lens, lens)                        # heads outside tokens


def test_views_past_32_bit_offsets():
    """Rows 2^20 elements apart: the last ones lie past 2^31 elements."""
    n = 2100
    g = torch.Generator(device="cuda").manual_seed(15)
    base = torch.empty(n, 1 << 20, dtype=torch.bfloat16, device="cuda")
    base[:, :1536] = torch.randn(n, 1536, generator=g, device="cuda").to(torch.bfloat16)
    base[:, 1536:1664] = float("nan")
    q, k, v = base[:, :1024].view(n, 8, 128), base[:, 1024:1280].view(n, 2, 128), \
        base[:, 1280:1536].view(n, 2, 128)
    check(q, k, v, [2000, 100], [2000, 100])


@pytest.mark.parametrize("d, dv", [(192, 128), (128, 128), (64, 64)])
def test_units_with_uneven_tiles_and_short_ones_in_turn(d, dv):
    """Pairs of Q tiles of which one ends a key tile early or has no token,
    followed on their SM by sequences of less than one key tile; the keys of
    some are more than the queries'.  Bit-identical when repeated."""
    lens_q = [200, 60, 129, 17, 256, 100, 90, 1] * 25
    lens_k = [200, 60, 500, 17, 256, 100, 700, 3] * 25
    case = tensors(lens_q, lens_k, 16, 16, d, dv, torch.bfloat16, seed=16)
    first = check(*case, lens_q, lens_k)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, check(*case, lens_q, lens_k)))


def test_many_sequences_and_long_ones():
    lens = [1 + (i * 37) % 90 for i in range(700)]
    check(*tensors(lens, lens, 4, 1, 64, 64, torch.bfloat16, seed=7), lens, lens)
    check(*tensors([4100], [4100], 2, 1, 128, 128, torch.bfloat16, seed=8), [4100], [4100])


def test_other_stream_and_repeat():
    lens = [300, 40]
    q, k, v = tensors(lens, lens, 8, 2, 128, 128, torch.bfloat16, seed=9)
    cu = torch.tensor([0, 300, 340], dtype=torch.int32, device="cuda")
    first = fa.prompt_attention(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = fa.prompt_attention(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)                 # no atomics: bit-identical


def test_captured_graph_sees_new_lengths():
    """Lengths are read on the device: a captured call follows new offsets."""
    lens = [100, 156]
    q, k, v = tensors(lens, lens, 4, 2, 64, 64, torch.bfloat16, seed=10)
    cu = torch.tensor([0, 100, 256], dtype=torch.int32, device="cuda")
    fa.prompt_attention(q, k, v, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.prompt_attention(q, k, v, cu)
    cu.copy_(torch.tensor([0, 31, 256], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want = fa.prompt_attention(q, k, v, cu)
    assert torch.equal(out, want)


def test_refusals():
    lens = [10, 20]
    q, k, v = tensors(lens, lens, 4, 2, 64, 64, torch.bfloat16)
    cu = torch.tensor([0, 10, 30], dtype=torch.int32, device="cuda")
    call = fa.prompt_attention
    with pytest.raises(fa.InvalidArgument):
        call(q, k.half(), v, cu)
    with pytest.raises(fa.InvalidArgument):
        call(q, k, v, cu.long())
    with pytest.raises(fa.InvalidArgument):
        call(q, k, v, cu.cpu())
    with pytest.raises(fa.InvalidArgument):
        call(q, k, v, cu, cu[:2])
    with pytest.raises(fa.InvalidArgument):
        call(q[:, :3], k, v, cu)
    with pytest.raises(fa.InvalidArgument):
        call(q, k[:, :, :32], v, cu)
    with pytest.raises(fa.InvalidArgument):
        call(q, k, v, cu, sm_scale=-1.0)
    with pytest.raises(fa.Unsupported):
        call(q.float(), k.float(), v.float(), cu)
    with pytest.raises(fa.Unsupported):
        call(*(torch.zeros(30, 1, 256, dtype=torch.bfloat16, device="cuda"),) * 3, cu)
    with pytest.raises(fa.Unsupported):
        call(*(torch.zeros(30, 1, 12, dtype=torch.bfloat16, device="cuda"),) * 3, cu)
    empty = call(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert empty.shape == (0, 4, 64)
