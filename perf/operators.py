"""Cases, plain forms and exact forms of the prompt attention and 4-bit cache operators.

``own`` false: ``run`` computes in elementary torch operations in 32 bits.  ``own`` true: ``run`` makes a user's calls of
``flagattention_b200``.  A case is a dict of plain values; sequence lengths follow from them (``lengths``).

Operators (the case's ``op``):

* ``prompt`` -- ``prompt_attention``: attention of packed prompts (sequence lengths ``lo`` .. ``hi``) over their own keys and
  ``ctx`` earlier keys per sequence; outputs the attention and the log-sum-exp.
* ``store``  -- ``append_kv_int4`` then ``read_kv_int4``: key / value rows go to their pages of the 4-bit cache and come back
  as the values that their codes stand for.
* ``decode`` -- ``paged_attention_int4``: one query token per sequence over a paged 4-bit cache.
"""

import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a short chat message: one prompt, latency of the call
        dict(name="prompt_short", op="prompt", batch=1, lo=37, hi=37, ctx=0, heads=64, kv_heads=8, dk=128, dv=128,
             causal=True, dtype="bf16"),
        # a serving step's waiting prompts packed together, single tokens to long ones
        dict(name="prompt_packed", op="prompt", batch=16, lo=1, hi=2048, ctx=0, heads=64, kv_heads=8, dk=128, dv=128,
             causal=True, dtype="bf16"),
        # one long document
        dict(name="prompt_long", op="prompt", batch=1, lo=8192, hi=8192, ctx=0, heads=64, kv_heads=8, dk=128, dv=128,
             causal=True, dtype="bf16"),
        # a small multi-head model in f16
        dict(name="prompt_d64_f16", op="prompt", batch=8, lo=300, hi=1501, ctx=0, heads=16, kv_heads=16, dk=64, dv=64,
             causal=True, dtype="f16"),
        # prompts of a latent-attention model: 128 + 64 rotary key dims, 128 value dims, every head with its own keys
        dict(name="prompt_latent", op="prompt", batch=2, lo=1000, hi=2048, ctx=0, heads=128, kv_heads=128, dk=192,
             dv=128, causal=True, dtype="bf16"),
        # the next chunk of a long prompt: few new tokens, many earlier keys
        dict(name="prompt_chunk", op="prompt", batch=1, lo=256, hi=256, ctx=16000, heads=64, kv_heads=8, dk=128,
             dv=128, causal=True, dtype="bf16"),
        # the new tokens of a decode step, one per sequence
        dict(name="store_step", op="store", tokens=64, kv_heads=8, d=128, group=64, page=16, dtype="bf16"),
        # the rows of a step's prompts
        dict(name="store_prompt", op="store", tokens=16383, kv_heads=8, d=128, group=64, page=16, dtype="bf16"),
        # one user
        dict(name="decode_one", op="decode", batch=1, lo=700, hi=700, heads=64, kv_heads=8, d=128, group=64, page=16,
             dtype="bf16"),
        # the batch of this repository's grouped-query benchmark, contexts of mixed lengths
        dict(name="decode_batch", op="decode", batch=32, lo=1000, hi=4096, heads=64, kv_heads=8, d=128, group=64,
             page=16, dtype="bf16"),
        # a few long documents
        dict(name="decode_long", op="decode", batch=8, lo=20001, hi=65536, heads=64, kv_heads=8, d=128, group=64,
             page=64, dtype="bf16"),
        # many short chats, small heads, wide groups, f16, finer scales
        dict(name="decode_d64_f16", op="decode", batch=64, lo=1, hi=4001, heads=64, kv_heads=4, d=64, group=32,
             page=32, dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = _cost(work(listed()[2]))
    while True:
        op = rng.choice(["prompt", "prompt", "store", "decode", "decode"])
        dtype = rng.choice(["bf16", "bf16", "f16"])
        if op == "prompt":
            hi = _log_int(rng, 1, 8192)
            dk, dv = rng.choice([(64, 64), (128, 128), (128, 128), (96, 96), (192, 128)])
            heads, kv = rng.choice([(64, 8), (32, 8), (16, 16), (24, 8), (40, 8), (64, 1)])
            c = dict(op=op, batch=_log_int(rng, 1, 32), lo=_log_int(rng, 1, hi), hi=hi,
                     ctx=rng.choice([0, 0, _log_int(rng, 1, 16000)]), heads=heads, kv_heads=kv, dk=dk, dv=dv,
                     causal=rng.random() < 0.75, dtype=dtype)
            # the plain form's padded scores stay within the largest listed case's
            if c["batch"] * heads * hi * (hi + c["ctx"]) > 64 * 8192 * 8192:
                continue
        elif op == "store":
            d = rng.choice([64, 128, 128, 256])
            c = dict(op=op, tokens=_log_int(rng, 1, 32768), kv_heads=rng.choice([1, 2, 4, 8, 16]), d=d,
                     group=rng.choice([g for g in (32, 64, 128) if d // 4 <= g <= d]), page=rng.choice([16, 32, 64, 128]),
                     dtype=dtype)
        else:
            d = rng.choice([64, 128, 128, 256])
            heads, kv = rng.choice([(64, 8), (32, 8), (16, 16), (24, 8), (40, 8), (64, 4), (32, 1)])
            hi = _log_int(rng, 1, 65536)
            c = dict(op=op, batch=_log_int(rng, 1, 64), lo=_log_int(rng, 1, hi), hi=hi, heads=heads, kv_heads=kv, d=d,
                     group=rng.choice([g for g in (32, 64, 128) if d // 4 <= g <= d]), page=rng.choice([16, 32, 64, 128]),
                     dtype=dtype)
            if c["batch"] * hi * kv * d > 8 * 65536 * 8 * 128:
                continue
        if _cost(work(c)) <= top:
            return c


def lengths(case):
    """New tokens (prompt) or context lengths (decode) per sequence: the first is ``hi``, the others spread over lo .. hi."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d" % case)
    return [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]


def _pairs(n, keys, causal):
    """Visible (query, key) pairs of n queries at the end of `keys` keys."""
    return n * keys - (n * (n - 1) // 2 if causal else 0)


def work(case):
    if case["op"] == "prompt":
        lens = lengths(case)
        q, keys = sum(lens), sum(lens) + case["ctx"] * len(lens)
        b = 2 * q * case["heads"] * (case["dk"] + case["dv"]) + 2 * keys * case["kv_heads"] * (case["dk"] + case["dv"])
        pairs = sum(_pairs(n, n + case["ctx"], case["causal"]) for n in lens)
        return {"bytes": b + 4 * q * case["heads"], "flops": 2 * (case["dk"] + case["dv"]) * case["heads"] * pairs}
    row = case["d"] + 8 * (case["d"] // case["group"])  # codes, scales and minima of one token and head, keys and values
    if case["op"] == "store":
        n = case["tokens"] * case["kv_heads"]
        return {"bytes": n * (2 * row + 8 * case["d"]) + 8 * case["tokens"], "flops": n * 2 * case["d"] * 8}
    keys = sum(lengths(case))
    b = keys * case["kv_heads"] * row + 4 * case["batch"] * case["heads"] * case["d"]
    return {"bytes": b + 4 * case["batch"] * case["heads"], "flops": 4 * case["d"] * case["heads"] * keys}


def _cost(w):
    return max(w["bytes"], w["flops"] / 50)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, n, heads, d, dtype):
    """Key rows (with the per-channel offsets that keys have) and value rows [n, heads, d]."""
    k = torch.randn(n, heads, d, generator=g, device="cuda") + 2 * torch.randn(heads, d, generator=g, device="cuda")
    v = torch.randn(n, heads, d, generator=g, device="cuda")
    return k.to(dtype), v.to(dtype)


def _offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).cuda()


def _pages(case, lens, g):
    """Block table [batch, width] over a shuffled pool, and the pool slot of every token in sequence order."""
    per = [-(-n // case["page"]) for n in lens]
    perm = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(per), dtype=torch.int32, device="cuda")
    table[torch.arange(max(per), device="cuda") < torch.tensor(per, device="cuda")[:, None]] = perm
    tok = torch.arange(max(lens), device="cuda")
    slots = table.long()[:, tok // case["page"]] * case["page"] + tok % case["page"]
    live = tok < torch.tensor(lens, device="cuda")[:, None]
    return table, slots[live], sum(per)


def prepare(case, seed):
    g, dtype = _generator(seed), _TYPES[case["dtype"]]
    if case["op"] == "prompt":
        lens = lengths(case)
        keys = [n + case["ctx"] for n in lens]
        q = torch.randn(sum(lens), case["heads"], case["dk"], generator=g, device="cuda").to(dtype)
        k = torch.randn(sum(keys), case["kv_heads"], case["dk"], generator=g, device="cuda").to(dtype)
        v = torch.randn(sum(keys), case["kv_heads"], case["dv"], generator=g, device="cuda").to(dtype)
        return dict(case=case, q=q, k=k, v=v, cu_q=_offsets(lens), cu_k=_offsets(keys), max_q=max(lens), max_k=max(keys))
    if case["op"] == "store":
        n = case["tokens"]
        k, v = _rows(g, n, case["kv_heads"], case["d"], dtype)
        blocks = -(-n // case["page"]) + 1
        slots = torch.randperm(blocks, generator=g, device="cuda")[torch.arange(n, device="cuda") // case["page"]]
        slots = slots * case["page"] + torch.arange(n, device="cuda") % case["page"]
        return dict(case=case, k=k, v=v, slots=slots, cache=_cache(case, blocks, dtype) if own else None)
    lens = lengths(case)
    table, slots, blocks = _pages(case, lens, g)
    k, v = _rows(g, sum(lens), case["kv_heads"], case["d"], dtype)
    s = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32).cuda(), max_len=max(lens),
             q=torch.randn(case["batch"], case["heads"], case["d"], generator=g, device="cuda").to(dtype))
    if own:  # the cache as a program has it after its prompts
        import flagattention_b200 as fa

        s["cache"] = fa.append_kv_int4(k, v, _cache(case, blocks, dtype), slots)
    else:  # the same rows as codes, minima and scales, by pool slot
        for name, x in (("k", k), ("v", v)):
            parts = _quantise(x, case["group"])
            pool = [p.new_zeros((blocks * case["page"],) + p.shape[1:]) for p in parts]
            for to, p in zip(pool, parts):
                to[slots] = p
            s[name] = pool
    return s


def _cache(case, blocks, dtype):
    import flagattention_b200 as fa

    return fa.Int4KVCache(blocks, case["kv_heads"], case["page"], case["d"], dtype=dtype, group_size=case["group"])


def run(state):
    if own:
        import flagattention_b200 as fa

        if state["case"]["op"] == "prompt":
            return fa.prompt_attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"],
                                       causal=state["case"]["causal"], return_lse=True)
        if state["case"]["op"] == "store":
            fa.append_kv_int4(state["k"], state["v"], state["cache"], state["slots"])
            return fa.read_kv_int4(state["cache"], state["slots"])
        return fa.paged_attention_int4(state["q"], state["cache"], state["lens"], state["table"], return_lse=True)
    return {"prompt": _prompt, "store": _store, "decode": _decode}[state["case"]["op"]](state)


# ---------------------------------------------------------------- plain forms


def _prompt(s):
    case, cu_q, cu_k = s["case"], s["cu_q"].long(), s["cu_k"].long()
    group = case["heads"] // case["kv_heads"]
    i, j = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    n, m = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    at_q = (cu_q[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    at_k = (cu_k[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = s["q"].float()[at_q].unflatten(2, (case["kv_heads"], group)).permute(0, 2, 3, 1, 4)  # [b, hk, g, i, d]
    k = s["k"].float()[at_k].permute(0, 2, 3, 1)[:, :, None]                                 # [b, hk, 1, d, j]
    v = s["v"].float()[at_k].permute(0, 2, 1, 3)[:, :, None]                                 # [b, hk, 1, j, d]
    p = (q.flatten(2, 3) @ k[:, :, 0]).mul_(case["dk"] ** -0.5).unflatten(2, (group, -1))
    hidden = (j >= m)[:, None, :]
    if case["causal"]:
        hidden = hidden | (j > i[:, None] + (m - n)[:, :, None])
    p.masked_fill_(hidden[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp(min=-3e38)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v[:, :, 0]).unflatten(2, (group, -1)) / total.clamp(min=1e-38)
    lse = (top + total.log())[..., 0]
    live = i < n
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[live]
    return o.to(s["q"].dtype), lse.permute(0, 3, 1, 2).flatten(2, 3)[live].t().contiguous()


def _quantise(x, group):
    """Codes 0 .. 15, minima and scales (in x's type) of groups of `group` dims."""
    x = x.unflatten(-1, (-1, group))
    lo, hi = x.amin(-1), x.amax(-1)
    scale = ((hi.float() - lo.float()) / 15).to(x.dtype)
    c = torch.round((x.float() - lo.float()[..., None]) / scale.float()[..., None]).clamp_(0, 15)
    return torch.where(scale[..., None] == 0, 0, c).to(torch.uint8).flatten(-2), lo, scale


def _values(codes, lo, scale):
    c = codes.float().unflatten(-1, (lo.shape[-1], -1))
    return (lo.float()[..., None] + c * scale.float()[..., None]).flatten(-2)


def _store(s):
    group, dtype = s["case"]["group"], s["k"].dtype
    return _values(*_quantise(s["k"], group)).to(dtype), _values(*_quantise(s["v"], group)).to(dtype)


def _decode(s):
    case, tok = s["case"], torch.arange(s["max_len"], device="cuda")
    at = s["table"].long()[:, tok // case["page"]] * case["page"] + tok % case["page"]
    k = _values(*(p[at] for p in s["k"])).permute(0, 2, 3, 1)                  # [b, hk, d, t]
    q = s["q"].float().unflatten(1, (case["kv_heads"], -1))                    # [b, hk, g, d]
    p = (q @ k) * case["d"] ** -0.5
    p.masked_fill_((tok >= s["lens"][:, None])[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp(min=-3e38)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = _values(*(p_[at] for p_ in s["v"])).permute(0, 2, 1, 3)                # [b, hk, t, d]
    o = (p @ v) / total.clamp(min=1e-38)
    return o.flatten(1, 2).to(s["q"].dtype), (top + total.log())[..., 0].flatten(1, 2)


# ------------------------------------------------- the definitions in 64 bits


def _attend64(q, k, v, scale, causal):
    """One sequence and kv head: q [rows of the group, n, dk], k [m, dk], v [m, dv] -> outputs, log-sum-exps."""
    n, m = q.shape[1], k.shape[0]
    s = torch.einsum("gid,jd->gij", q, k) * scale
    if causal:
        s[:, torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)] = -math.inf
    lse = torch.logsumexp(s, -1)
    return torch.einsum("gij,jd->gid", torch.softmax(s, -1), v), lse


def _stored64(x, group):
    """The values that rows x stand for in 4 bits: lo + scale * code, scale held in x's type."""
    y = x.double().unflatten(-1, (-1, group))
    lo = y.min(-1, keepdim=True).values
    scale = ((y.max(-1, keepdim=True).values - lo) / 15).to(x.dtype).double()
    code = torch.where(scale > 0, ((y - lo) / scale).round().clamp(0, 15), torch.zeros_like(y))
    return (lo + scale * code).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _stored64(s["k"], case["group"]), _stored64(s["v"], case["group"])
    lens, heads, hk = lengths(case), case["heads"], case["kv_heads"]
    if case["op"] == "prompt":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        keys, dk, dv, causal = [n + case["ctx"] for n in lens], case["dk"], case["dv"], case["causal"]
    else:  # the same generator gives the rows that prepare() stored, in sequence order
        g = _generator(seed)
        _pages(case, lens, g)
        k, v = (_stored64(x, case["group"]) for x in _rows(g, sum(lens), hk, case["d"], _TYPES[case["dtype"]]))
        q, keys, lens, dk, dv, causal = s["q"].double(), lens, [1] * len(lens), case["d"], case["d"], False
    del s
    out, lse = q.new_zeros(sum(lens), heads, dv), q.new_zeros(heads, sum(lens))
    a, b, per = 0, 0, heads // hk
    for n, m in zip(lens, keys):
        for h in range(hk):
            mine = slice(h * per, (h + 1) * per)
            o, l = _attend64(q[a:a + n, mine].transpose(0, 1), k[b:b + m, h], v[b:b + m, h], dk ** -0.5, causal)
            out[a:a + n, mine], lse[mine, a:a + n] = o.transpose(0, 1), l
        a, b = a + n, b + m
    return out, lse if case["op"] == "prompt" else lse.t().contiguous()
