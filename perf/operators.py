"""Cases of the serving operators around a 4-bit key/value cache, for timing.

Four operators of a prompt and of the decode tokens that follow it:

  rope     bias, per-head norms of queries and keys and the position rotation
           of a batch of tokens, in one pass        attention.qk_norm_rope
  cache    keys and values of tokens quantised into a paged 4-bit cache, and
           read back      attention.kv_append_q4, attention.kv_read_q4
  decode   one query token for each sequence over the paged 4-bit cache
                                             attention.attention_decode_q4
  prompt   causal attention of whole prompts, packed, with grouped heads
                                               attention.attention_prefill

`run` computes them in elementary torch operations where `own` is false, and
through the package's entry points where it is true.

The 4-bit cache is a uint8 tensor (pages, kv_heads, page_size / 16, 20 * dim):
blocks of 16 tokens of one head.  A token's channels are quantised in groups
of 32 with an fp16 step d and an fp16 offset m, value = d * n + m, n in 0..15.
A block holds, in bytes (NG = dim / 32 groups, nibble i of a word is bits
4i..4i+3):
  K nibbles  (16 tokens, 4, NG) words; word (q, j) has channels 32 j + 8 q ..
  V nibbles  (dim / 8, 16 tokens) words; word w has channels 8 w ..
  K steps (NG, 16), K offsets (16, NG), V steps (NG, 16), V offsets (NG, 16)
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- the cases ------------------------------------------------------------------
def listed():
    return [
        # one decode token of a Qwen2-7B-shaped layer: the smallest call, biases, fp32 as the decoder computes
        {"name": "rope token 28x4", "op": "rope", "tokens": 1, "heads": 28, "kv_heads": 4, "dim": 128, "rot": 128,
         "in": "fp32", "out": "fp32", "bias": True, "norm": False, "interleaved": False, "longest": 4096},
        # a few hundred tokens of a running batch: norms of queries and keys, half of the head rotated, pairs adjacent
        {"name": "rope batch norm", "op": "rope", "tokens": 389, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "in": "bf16", "out": "bf16", "bias": False, "norm": True, "interleaved": True, "longest": 131072},
        # a whole prompt of a Llama-3-70B-shaped layer: fp32 projections to the 16-bit queries, keys and values
        {"name": "rope prompt 64x8", "op": "rope", "tokens": 8192, "heads": 64, "kv_heads": 8, "dim": 128, "rot": 128,
         "in": "fp32", "out": "bf16", "bias": False, "norm": False, "interleaved": False, "longest": 8192},
        # the new token of each of 32 sequences
        {"name": "cache token x32", "op": "cache", "tokens": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "fp32", "contiguous": False},
        # a prompt of odd length, small heads, fp32
        {"name": "cache prompt 1531", "op": "cache", "tokens": 1531, "kv_heads": 4, "dim": 64, "page": 16,
         "dtype": "fp32", "contiguous": True},
        # long prompts of a Llama-3-70B-shaped layer
        {"name": "cache prompts 65536", "op": "cache", "tokens": 65536, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "contiguous": True},
        # one sequence of a Qwen2-7B-shaped layer at 4097 positions, fp32 queries as the decoder's
        {"name": "decode 28x4 4097", "op": "decode", "batch": 1, "longest": 4097, "heads": 28, "kv_heads": 4,
         "dim": 128, "page": 64, "dtype": "fp32", "mix": 1},
        # a serving batch of a Llama-3-70B-shaped layer: 128 sequences from a token to 8192, small pages
        {"name": "decode 64x8 batch 128", "op": "decode", "batch": 128, "longest": 8192, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "mix": 2},
        # few very long contexts
        {"name": "decode 32x8 131071", "op": "decode", "batch": 5, "longest": 131071, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "fp16", "mix": 3},
        # a short prompt of a Qwen2-7B-shaped layer: latency
        {"name": "prompt 28x4 77", "op": "prompt", "batch": 1, "longest": 77, "past": 0, "pad": 0, "heads": 28,
         "kv_heads": 4, "dim": 128, "dtype": "bf16", "causal": True, "mix": 4},
        # packed prompts of many lengths that go on behind cached tokens, small heads, padded rows at the end
        {"name": "prompts packed 17", "op": "prompt", "batch": 17, "longest": 1000, "past": 300, "pad": 37,
         "heads": 32, "kv_heads": 8, "dim": 64, "dtype": "fp16", "causal": True, "mix": 5},
        # a long prompt of a Llama-3-70B-shaped layer
        {"name": "prompt 64x8 8192", "op": "prompt", "batch": 1, "longest": 8192, "past": 0, "pad": 0, "heads": 64,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "causal": True, "mix": 6},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "decode", "prompt"])
    dim = rng.choice([64, 128, 128])
    heads, kv_heads = rng.choice([(28, 4), (64, 8), (32, 8), (14, 2), (16, 16), (24, 8), (32, 2)])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        return {"op": op, "tokens": _log(rng, 1, 8192 * 64 * 128 // (heads * dim)), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "in": dtype,
                "out": rng.choice([dtype, "bf16"]), "bias": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "interleaved": rng.random() < 0.5, "longest": rng.choice([4096, 32768, 131072])}
    if op == "cache":
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        tokens = _log(rng, 1, 65536 * 8 * 128 // (kv_heads * dim) // (2 if dtype == "fp32" else 1))
        contiguous = rng.random() < 0.7
        return {"op": op, "tokens": min(tokens, 131072 if contiguous else 2048), "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "contiguous": contiguous}
    if op == "decode":
        batch = _log(rng, 1, 128)
        return {"op": op, "batch": batch, "longest": _log(rng, 1, min(131071, 8 * 524288 // (batch * kv_heads))),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["fp32", "bf16", "fp16"]), "mix": rng.randrange(1 << 16)}
    batch = _log(rng, 1, 24)
    return {"op": op, "batch": batch, "longest": _log(rng, 1, 8192 // batch),
            "past": rng.choice([0, 0, 64, 300]), "pad": rng.choice([0, 0, 5, 130]), "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "fp16"]), "causal": rng.random() < 0.8,
            "mix": rng.randrange(1 << 16)}


def _lengths(case):
    """The sequences' lengths: the longest, and the others spread over the logarithm below it."""
    r = random.Random(case["mix"])
    rest = [_log(r, 1, case["longest"]) for _ in range(case["batch"] - 1)]
    n = [case["longest"]] + rest
    r.shuffle(n)
    return n


def _prompt_lengths(case):
    """(queries, keys) of each sequence: keys are the cached tokens before the prompt and the prompt itself."""
    q = _lengths(case)
    r = random.Random(case["mix"] + 1)
    return q, [n + r.randrange(case["past"] + 1) for n in q]


def work(case):
    op, dim = case["op"], case["dim"]
    if op == "rope":
        rows = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * dim
        return {"bytes": rows * (_BYTES[case["in"]] + _BYTES[case["out"]]) + case["tokens"] * (case["rot"] + 1) * 4,
                "flops": rows * 6}
    if op == "cache":
        n = 2 * case["tokens"] * case["kv_heads"] * dim
        return {"bytes": 2 * n * _BYTES[case["dtype"]] + 2 * n * 5 // 8 + 16 * case["tokens"], "flops": n * 8}
    if op == "decode":
        tokens, rows = sum(_lengths(case)), case["batch"] * case["heads"] * dim
        return {"bytes": tokens * case["kv_heads"] * dim * 5 // 4 + 2 * rows * _BYTES[case["dtype"]],
                "flops": 4 * tokens * case["heads"] * dim}
    nq, nk = _prompt_lengths(case)
    pairs = sum(q * k - (q * (q - 1) // 2 if case["causal"] else 0) for q, k in zip(nq, nk))
    return {"bytes": 2 * dim * (2 * sum(nq) * case["heads"] + 2 * sum(nk) * case["kv_heads"]),
            "flops": 4 * pairs * case["heads"] * dim}


# ---- inputs -----------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=dev) * std

    op, dim = case["op"], case["dim"]
    s = {"case": case}
    if op == "rope":
        t, nh, nkv, rot = case["tokens"], case["heads"], case["kv_heads"], case["rot"]
        n = (nh + 2 * nkv) * dim
        s["qkv"] = normal(t, n, std=2.0).to(_DTYPES[case["in"]])
        s["bias"] = normal(n, std=0.5) if case["bias"] else None
        s["q_norm"] = 1 + normal(dim, std=0.1) if case["norm"] else None
        s["k_norm"] = 1 + normal(dim, std=0.1) if case["norm"] else None
        # angles in 64 bits: far positions lose the fast pairs' phase in 32
        inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        angle = torch.arange(case["longest"], dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if t <= 512:  # tokens of many sequences, each at a position of its own
            s["pos"] = torch.randint(0, case["longest"], (t,), generator=g, device=dev, dtype=torch.int32)
        else:
            s["pos"] = torch.arange(t, device=dev, dtype=torch.int32) % case["longest"]
        out = _DTYPES[case["out"]]
        s["out"] = tuple(torch.zeros((t, h, dim), dtype=out, device=dev) for h in (nh, nkv, nkv))
        return s
    if op == "cache":
        t, nkv, page = case["tokens"], case["kv_heads"], case["page"]
        dtype = _DTYPES[case["dtype"]]
        # keys have a few channels far larger than the rest, values have not
        channel = torch.ones(dim, device=dev)
        channel[:: max(1, dim // 4)] = 8.0
        s["k"] = (normal(t, nkv, dim) * channel + 0.5 * channel).to(dtype)
        s["v"] = normal(t, nkv, dim).to(dtype)
        if case["contiguous"]:  # a prompt: its pages are anywhere, filled one after the other
            pages = -(-t // page)
            order = torch.randperm(pages, generator=g, device=dev)
            i = torch.arange(t, device=dev)
            s["slots"] = order[i // page] * page + i % page
        else:  # a token of each sequence: each in a page of its own
            pages = t
            s["slots"] = torch.arange(t, device=dev) * page + torch.randint(0, page, (t,), generator=g, device=dev)
        s["cache"] = torch.zeros((pages, nkv, page // 16, 20 * dim), dtype=torch.uint8, device=dev)
        s["out"] = (torch.zeros((t, nkv, dim), dtype=dtype, device=dev),
                    torch.zeros((t, nkv, dim), dtype=dtype, device=dev))
        return s
    nh, nkv = case["heads"], case["kv_heads"]
    dtype = _DTYPES[case["dtype"]]
    if op == "decode":
        page, n = case["page"], _lengths(case)
        need = [-(-x // page) for x in n]
        pages = sum(need)
        groups = dim // 32
        s["q"] = normal(case["batch"], nh, dim).to(dtype)
        cache = torch.randint(0, 256, (pages, nkv, page // 16, 20 * dim), generator=g, device=dev, dtype=torch.uint8)
        scales = cache[..., 16 * dim:].view(torch.float16).unflatten(-1, (4, 16 * groups))
        step = 0.1 + 0.3 * torch.rand(scales.shape[:-2] + (2, groups, 16), generator=g, device=dev)
        offset = -step * (6 + 3 * torch.rand(step.shape, generator=g, device=dev))
        scales[..., 0, :] = step[..., 0, :, :].flatten(-2).half()
        scales[..., 1, :] = offset[..., 0, :, :].transpose(-1, -2).flatten(-2).half()
        scales[..., 2, :] = step[..., 1, :, :].flatten(-2).half()
        scales[..., 3, :] = offset[..., 1, :, :].flatten(-2).half()
        s["cache"] = cache
        order = torch.randperm(pages, generator=g, device=dev).int()
        table = torch.zeros((case["batch"], max(need)), dtype=torch.int32, device=dev)
        at = 0
        for b, c in enumerate(need):
            table[b, :c] = order[at:at + c]
            at += c
        s["table"], s["lengths"] = table, torch.tensor(n, dtype=torch.int32, device=dev)
        s["out"] = torch.zeros((case["batch"], nh, dim), dtype=dtype, device=dev)
        return s
    nq, nk = _prompt_lengths(case)
    tq, tk = sum(nq) + case["pad"], sum(nk) + case["pad"]
    s["q"] = normal(tq, nh, dim, std=1.5).to(dtype)
    s["k"], s["v"] = normal(tk, nkv, dim).to(dtype), normal(tk, nkv, dim).to(dtype)
    ends = [[sum(x[:i]) for i in range(len(x) + 1)] for x in (nq, nk)]
    s["cu_q"], s["cu_k"] = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ends)
    s["out"] = torch.zeros((tq, nh, dim), dtype=dtype, device=dev)
    return s


# ---- the 4-bit cache in elementary operations ----------------------------------------
def _to_half_grid(x):
    """64-bit x >= 0 at the nearest fp16 value (ties to even), at most 65504."""
    _, e = torch.frexp(x)
    ulp = torch.ldexp(torch.ones_like(x), (e - 11).clamp(min=-24))
    return (torch.round(x / ulp) * ulp).clamp(max=65504.0)


def _quantise(x):
    """(nibbles, steps, offsets) of x (..., dim): by definition in exact arithmetic, so in 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    low, high = g.amin(-1), g.amax(-1)
    offset = low.float().clamp(-65504.0, 65504.0).half()
    step = _to_half_grid(((high - offset.double()) / 15).clamp(min=0)).half()
    d = step.double()[..., None]
    n = torch.round((g - offset.double()[..., None]) / torch.where(d > 0, d, torch.ones_like(d))).clamp(0, 15)
    n = torch.where(d > 0, n, torch.zeros_like(n))
    bad = ~torch.isfinite(g).all(-1)
    offset = torch.where(bad, torch.full_like(offset, float("nan")), offset)
    step = torch.where(bad, torch.zeros_like(step), step)
    n = torch.where(bad[..., None], torch.zeros_like(n), n)
    return n.flatten(-2).to(torch.uint8), step, offset


def _parts(cache):
    """Views of a cache's parts: K bytes (.., 16, 4, NG, 4), V bytes (.., dim / 8, 16, 4) and the scales."""
    dim = cache.shape[-1] // 20
    ng, kb = dim // 32, 8 * dim
    k = cache[..., :kb].unflatten(-1, (16, 4, ng, 4))
    v = cache[..., kb:2 * kb].unflatten(-1, (dim // 8, 16, 4))
    sc = cache[..., 2 * kb:].view(torch.float16).unflatten(-1, (4, 16 * ng))
    return (k, v, sc[..., 0, :].unflatten(-1, (ng, 16)), sc[..., 1, :].unflatten(-1, (16, ng)),
            sc[..., 2, :].unflatten(-1, (ng, 16)), sc[..., 3, :].unflatten(-1, (ng, 16)))


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)


def _bytes(n):
    n = n.unflatten(-1, (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def _write(cache, k, v, slots):
    page = cache.shape[2] * 16
    p, c, t = slots // page, slots % page // 16, slots % 16
    kn, kd, km = _quantise(k)
    vn, vd, vm = _quantise(v)
    pk, pv, pkd, pkm, pvd, pvm = _parts(cache)
    ng = kd.shape[-1]
    pk[p, :, c, t] = _bytes(kn.unflatten(-1, (ng, 4, 8)).transpose(-3, -2))
    pv[p, :, c, :, t] = _bytes(vn.unflatten(-1, (-1, 8)))
    pkd[p, :, c, :, t], pkm[p, :, c, t] = kd, km
    pvd[p, :, c, :, t], pvm[p, :, c, :, t] = vd, vm


def _read(cache, p, c, t, wide):
    """K and V of the tokens (p, c, t) as (.., kv_heads, dim) in the type `wide`."""
    pk, pv, pkd, pkm, pvd, pvm = _parts(cache)
    kn = _nibbles(pk[p, :, c, t]).transpose(-3, -2).flatten(-2)
    vn = _nibbles(pv[p, :, c, :, t]).unflatten(-2, (-1, 4)).flatten(-2)
    k = kn.to(wide) * pkd[p, :, c, :, t].to(wide)[..., None] + pkm[p, :, c, t].to(wide)[..., None]
    v = vn.to(wide) * pvd[p, :, c, :, t].to(wide)[..., None] + pvm[p, :, c, :, t].to(wide)[..., None]
    return k.flatten(-2), v.flatten(-2)


def _read_sequences(cache, table, wide):
    """K and V of whole sequences, (batch, kv_heads, positions, dim)."""
    blocks = cache[table.long()]  # (batch, pages, heads, blocks, bytes)
    pk, pv, pkd, pkm, pvd, pvm = _parts(blocks)
    k = _nibbles(pk).transpose(-3, -2).flatten(-2).to(wide)  # (.., 16, NG, 32)
    k = k * pkd.transpose(-1, -2).to(wide)[..., None] + pkm.to(wide)[..., None]
    v = _nibbles(pv).unflatten(-3, (-1, 4)).transpose(-3, -2).transpose(-4, -3).flatten(-2)  # (.., 16, NG, 32)
    v = v.to(wide) * pvd.transpose(-1, -2).to(wide)[..., None] + pvm.transpose(-1, -2).to(wide)[..., None]
    return tuple(x.flatten(-2).permute(0, 2, 1, 3, 4, 5).flatten(2, 4) for x in (k, v))


# ---- one pass ---------------------------------------------------------------------
def _rope(s, wide):
    c = s["case"]
    nh, nkv, dim, rot = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s["qkv"].to(wide)
    if s["bias"] is not None:
        x = x + s["bias"].to(wide)
    q, k, v = x.unflatten(-1, (-1, dim)).split((nh, nkv, nkv), dim=1)
    cos, sin = (s[n][s["pos"].long()].to(wide)[:, None] for n in ("cos", "sin"))

    def turn(h, w):
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.to(wide)
        r = h[..., :rot]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((r, h[..., rot:]), dim=-1)

    return turn(q, s["q_norm"]), turn(k, s["k_norm"]), v


def _decode(s):
    c = s["case"]
    nkv, dim = c["kv_heads"], c["dim"]
    k, v = _read_sequences(s["cache"], s["table"], torch.float32)
    q = s["q"].float().unflatten(1, (nkv, -1)) * (1.0 / math.sqrt(dim))
    p = q @ k.transpose(-1, -2)  # (batch, kv_heads, group, positions)
    out = torch.arange(p.shape[-1], device=p.device) >= s["lengths"][:, None]
    p = p.masked_fill_(out[:, None, None], float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    return ((p @ v) / p.sum(-1, keepdim=True)).flatten(1, 2).to(s["q"].dtype)


def _seen(cu_q, cu_k, tq, tk, causal):
    """(tq, tk): whether a query sees a key."""
    iq, ik = torch.arange(tq, device=cu_q.device), torch.arange(tk, device=cu_q.device)
    bq, bk = (torch.searchsorted(cu, i.int(), right=True) - 1 for cu, i in ((cu_q, iq), (cu_k, ik)))
    last = cu_q.shape[0] - 1
    seen = (bq[:, None] == bk) & (bq < last)[:, None]
    if causal:  # the last query sees the last key
        end_q, end_k = cu_q[1:].long(), cu_k[1:].long()
        from_end_q = end_q[bq.clamp(max=last - 1)] - iq
        from_end_k = end_k[bk.clamp(max=last - 1)] - ik
        seen &= from_end_k >= from_end_q[:, None]
    return seen


def _prompt(s):
    c = s["case"]
    nkv, dim, dtype = c["kv_heads"], c["dim"], s["q"].dtype
    tq, tk = s["q"].shape[0], s["k"].shape[0]
    q = (s["q"].float() * (1.0 / math.sqrt(dim))).unflatten(1, (nkv, -1)).permute(1, 2, 0, 3)
    k, v = (s[n].float().transpose(0, 1) for n in ("k", "v"))
    hidden = ~_seen(s["cu_q"], s["cu_k"], tq, tk, c["causal"])
    p = (q.flatten(1, 2) @ k.transpose(-1, -2)).unflatten(1, (-1, tq))
    p = p.masked_fill_(hidden, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(1, 2) @ v).unflatten(1, (-1, tq)) / torch.where(total > 0, total, torch.ones_like(total))
    return o.flatten(0, 1).transpose(0, 1).to(dtype).contiguous()


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        from flatrun_b200 import attention

        if op == "rope":
            return attention.qk_norm_rope(s["qkv"], c["heads"], c["kv_heads"], s["cos"], s["sin"], s["pos"],
                                          bias=s["bias"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
                                          interleaved=c["interleaved"], out=s["out"])
        if op == "cache":
            attention.kv_append_q4(s["cache"], s["k"], s["v"], s["slots"])
            return attention.kv_read_q4(s["cache"], s["slots"], out=s["out"])
        if op == "decode":
            return attention.attention_decode_q4(s["q"], s["cache"], s["table"], s["lengths"], out=s["out"])
        return attention.attention_prefill(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=c["causal"],
                                           out=s["out"])
    if op == "rope":
        dtype = _DTYPES[c["out"]]
        return tuple(x.to(dtype) for x in _rope(s, torch.float32))
    if op == "cache":
        slots, page = s["slots"], c["page"]
        _write(s["cache"], s["k"], s["v"], slots)
        k, v = _read(s["cache"], slots // page, slots % page // 16, slots % 16, torch.float32)
        return k.to(s["k"].dtype), v.to(s["v"].dtype)
    if op == "decode":
        return _decode(s)
    return _prompt(s)


# ---- the definitions in 64 bits ----------------------------------------------------------
def _exact_rope(s):
    c = s["case"]
    nh, nkv, dim, rot = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s["qkv"].double() + (s["bias"].double() if s["bias"] is not None else 0.0)
    x = x.reshape(c["tokens"], nh + 2 * nkv, dim)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None, :]
    first = torch.arange(0, rot, 2, device=x.device) if c["interleaved"] else torch.arange(rot // 2, device=x.device)
    second = first + (1 if c["interleaved"] else rot // 2)
    got = []
    for lo, hi, w in ((0, nh, s["q_norm"]), (nh, nh + nkv, s["k_norm"])):
        h = x[:, lo:hi].clone()
        if w is not None:
            h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / dim + 1e-6) * w.double()
        z = torch.complex(h[..., first], h[..., second]) * turn
        h[..., first], h[..., second] = z.real, z.imag
        got.append(h)
    return got[0], got[1], x[:, nh + nkv:]


def _exact_cache(x):
    """What each value of x (tokens, heads, dim) stands for after 4 bits, from the definition."""
    t, h, dim = x.shape
    g = x.double().reshape(t * h * (dim // 32), 32)
    m = g.min(1).values.float().clamp(-65504, 65504).half().double()
    d = (g.max(1).values - m).clamp(min=0) / 15
    scale = torch.exp2(torch.floor(torch.log2(d.clamp(min=2.0 ** -14))))  # the binade's fp16 spacing, 1024 to a binade
    d = (torch.round(d / scale * 1024) / 1024 * scale).clamp(max=65504)
    n = ((g - m[:, None]) / d.clamp(min=2.0 ** -24)[:, None]).round().clamp(0, 15)
    return (n * d[:, None] + m[:, None]).reshape(t, h, dim)


def _exact_attention(q, k, v, hidden):
    """q (rows, dim), k and v (keys, dim), hidden (rows, keys) or None, in 64 bits."""
    a = (q.double() @ k.double().T) / math.sqrt(q.shape[-1])
    if hidden is not None:
        a.masked_fill_(hidden, -math.inf)
    a = torch.nan_to_num(torch.softmax(a, dim=-1), nan=0.0)
    return a @ v.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_rope(s)
    if op == "cache":
        return _exact_cache(s["k"]), _exact_cache(s["v"])
    nkv, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // nkv
    if op == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        page = case["page"]
        for b, n in enumerate(s["lengths"].tolist()):
            i = torch.arange(n, device=out.device)
            k, v = _read(s["cache"], s["table"][b].long()[i // page], i % page // 16, i % 16, torch.float64)
            for h in range(nkv):
                rows = slice(h * group, (h + 1) * group)
                out[b, rows] = _exact_attention(s["q"][b, rows], k[:, h], v[:, h], None)
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(case["batch"]):
        nq, nk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        hidden = None
        if case["causal"]:
            hidden = torch.ones((nq, nk), dtype=torch.bool, device=out.device).triu(nk - nq + 1)
        for h in range(case["heads"]):
            rows, keys = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
            out[rows, h] = _exact_attention(s["q"][rows, h], s["k"][keys, h // group], s["v"][keys, h // group],
                                            hidden)
    return out
