"""Decode attention over the 4-bit cache at the ends of the numbers' range (GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flatrun_b200 import attention as A
import q4_restated as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lens", [[1, 0, 40, 700], [30000, 3, 0]])  # the second: pieces of warps, CTAs, and the join of both
def test_scores_of_minus_infinity(dtype, lens):
    """Queries of -1e37 over keys of 30: every score is -inf, and the softmax 0 / 0.  No token gives zeros, hidden pages
    too; a token of score 0 among them takes all the weight, wherever it lies."""
    nh, nkv, hd, page = 4, 2, 64, 16
    need = [-(-n // page) for n in lens]
    cache = A.kv_cache_q4(sum(need), page, nkv, hd)
    table = torch.full((len(lens) + 1, max(need)), -1, dtype=torch.int32)  # (the last sequence: hidden pages alone)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = torch.arange(at, at + c)
        at += c
    slots = torch.arange(at * page, device="cuda")
    v = torch.randn((at * page, nkv, hd), device="cuda")
    A.kv_append_q4(cache, torch.full_like(v, 30.0), v, slots)
    table = table.cuda()
    n = torch.tensor([*lens, 16], dtype=torch.int32, device="cuda")
    q = torch.full((len(lens) + 1, nh, hd), -1e37, device="cuda").to(DT[dtype])
    some = torch.tensor([m > 0 for m in lens] + [False], device="cuda")
    for h in range(nh):  # (other heads have finite scores)
        x = torch.zeros_like(q)
        x[:, h] = q[:, h]
        got = A.attention_decode_q4(x, cache, table, n)
        assert bool(torch.isnan(got[some, h]).all())
        assert not bool(torch.isnan(got).any(-1)[:, [i for i in range(nh) if i != h]].any())
        assert not got[~some].any()
    for b, m in enumerate(lens):
        for t in {0, m // 2, m - 1} if m else ():
            slot = table[b, t // page].long()[None] * page + t % page
            A.kv_append_q4(cache, torch.zeros(1, nkv, hd, device="cuda"), v[slot], slot)
            got = A.attention_decode_q4(q, cache, table, n)[b]
            ref = A.kv_read_q4(cache, slot)[1][0].repeat_interleave(nh // nkv, 0)
            # the weight is 1: the value's own roundings (n - 8, m + 8 d: a few of its terms' sizes) and the type's
            size = 4 * v.abs().max()
            half = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -11}[dtype]
            bound = 8 * half * size + (2.0 ** -8 if dtype == "bf16" else 0) * ref.abs()
            assert bool(((got.float() - ref).abs() <= bound).all())
            A.kv_append_q4(cache, torch.full((1, nkv, hd), 30.0, device="cuda"), v[slot], slot)


E32 = 2.0 ** -24
HALF_TYPE = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _attend(scores, values, dtype, nh, hd, page=16, seed=0):
    """Decode attention of `nh` query heads over one KV head, where token t has the score scores[t] (about: in the cache's 4
    bits) and the values values[t]; the result and its bound against 64 bits.

    Scores: 40 roundings of the products' sizes and 4 of exp2's argument: delta.  Weights and steps rounded to fp16 for the
    16-bit types (twice 2^-11, of |d (n - 8)| + |m + 8 d| or less), 64 roundings in fp32; the type's own.  No floor: a token's
    share counts however large the others' values are.  (Weights are above 2^-25 of the largest in these tests.)"""
    t = len(scores)
    rng = np.random.default_rng(seed)
    pages = -(-t // page) + 1
    cache = torch.from_numpy(rng.integers(0, 256, (pages, 1, page // 16, 20 * hd), dtype=np.uint8)).cuda()
    order = rng.permutation(pages)[:-(-t // page)].astype(np.int32)
    k = np.zeros((t, 1, hd), np.float32)
    k[:, 0, 40] = scores
    slots = order[np.arange(t) // page].astype(np.int64) * page + np.arange(t) % page
    A.kv_append_q4(cache, torch.from_numpy(k).cuda(), torch.from_numpy(values[:, None].astype(np.float32)).cuda(),
                   torch.from_numpy(slots).cuda())
    q = np.zeros((1, nh, hd), np.float32)
    q[0, :, 40] = 1 + np.arange(nh) / 16  # exact in all types
    got = A.attention_decode_q4(torch.from_numpy(q).cuda().to(DT[dtype]), cache, torch.from_numpy(order[None]).cuda(),
                                torch.tensor([t], dtype=torch.int32).cuda(), scale=1.0)
    with np.errstate(all="ignore"):
        kk, vv, _, vs = R.unpack(cache.cpu().numpy())
        vs = np.maximum(vs, R.middle_sizes(cache.cpu().numpy()))
    kk, vv, vs = (x[slots // page, 0, slots % page] for x in (kk, vv, vs))
    s = q[0].astype(np.float64) @ kk.T
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    o = p @ vv
    delta = 44 * E32 * np.abs(s).max(-1, keepdims=True) + 4 * E32
    step = 64 * E32 if dtype == "fp32" else 2 * 2.0 ** -11 + 64 * E32
    bound = (np.expm1(2 * delta) + step) * (p @ vs) + HALF_TYPE[dtype] * np.abs(o) + (2.0 ** -25 if dtype == "fp16" else 0)
    return got[0].double().cpu().numpy(), o, bound


def _check(got, o, bound):
    bad = ~(np.abs(got - o) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], o[bad][:4], bound[bad][:4])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens,at", [(8, 3), (32, 0), (700, 0), (700, 350), (700, 695), (9000, 8000)])
@pytest.mark.parametrize("size", [40.0, 1e3, 6e4])
def test_one_large_token_of_small_weight(dtype, hd, tokens, at, size):
    """Values of 0.3 and a token of far larger ones whose score is 16 powers of two below the others'."""
    rng = np.random.default_rng(tokens + at)
    v = 0.3 * rng.standard_normal((tokens, hd))
    v[at] *= size / 0.3 / 3
    s = -0.05 * rng.random(tokens)
    s[at] = -16 * np.log(2)
    _check(*_attend(s, np.clip(v, -6.4e4, 6.4e4), dtype, 3, hd))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("hd,tokens", [(64, 20), (128, 64), (128, 500)])
@pytest.mark.parametrize("large", [1.0, 2e4])
def test_one_large_group_beside_small_ones(dtype, hd, tokens, large):
    """In every token one group of 32 channels is 10^7 times as large as another."""
    rng = np.random.default_rng(tokens)
    v = rng.standard_normal((tokens, hd)) * np.repeat(np.resize([large, large * 1e-7], hd // 32), 32)
    _check(*_attend(-3 * rng.random(tokens), v, dtype, 8, hd))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("first,rest", [(1e-4, 1e3), (1e3, 1e-4), (1e4, 1e4), (0.0, 1.0), (1.0, 0.0), (1e-6, 1e-6)])
def test_values_that_change_their_size(dtype, first, rest):
    """The first tokens' values far smaller or larger than the others', or zeros; one size for all."""
    rng = np.random.default_rng(5)
    v = rng.standard_normal((3000, 64))
    v[:45] *= first
    v[45:] *= rest
    if dtype == "fp16":
        v *= 0.25
    _check(*_attend(-8 * rng.random(3000), v, dtype, 2, 64))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_small_weights_of_large_values(dtype):
    """One token takes most of the weight; 20000 of 2^-18 each add a tenth, with values of 1e4."""
    rng = np.random.default_rng(6)
    v = 1e4 * rng.standard_normal((20000, 128))
    s = -18 * np.log(2) * np.ones(20000)
    s[11] = 0.0
    _check(*_attend(s, v, dtype, 4, 128))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_constant_values(dtype):
    """Groups without a step: every value is its offset."""
    v = np.repeat(np.array([[1.5, -3.0, 0.0, 1000.0]]), 32, axis=1).repeat(100, axis=0)
    got, o, bound = _attend(np.linspace(-4, 0, 100), v, dtype, 2, 128)
    _check(got, o, bound)
    assert not got[:, 64:96].any()
