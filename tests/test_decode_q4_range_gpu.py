"""Decode attention over the 4-bit cache at the ends of the numbers' range (GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flatrun_b200 import attention as A

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
