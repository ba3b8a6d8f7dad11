"""The serving operators against their restatement in 64 bits (GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flatrun_b200 import attention as A
import q4_restated as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E32 = 2.0 ** -24


def _rand(rng, shape, dtype, std=1.0):
    """A tensor on the GPU, and its values."""
    t = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(DT[dtype]).cuda()
    return t, _np(t)


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, bound):
    got = _np(got)
    assert got.shape == ref.shape
    bad = ~(np.abs(got - ref) <= bound) & ~(np.isnan(ref) & np.isnan(got))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], ref[bad][:3],
                           np.broadcast_to(bound, ref.shape)[bad][:3])


# ---- rotation -------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,nh,nkv,hd,rot,inter,norm,bias,tin,tout", [
    (1, 28, 4, 128, 128, False, False, True, "fp32", "fp32"),
    (7, 4, 2, 64, 64, True, True, True, "fp32", "fp32"),
    (5, 3, 1, 80, 40, False, True, False, "bf16", "bf16"),
    (6, 2, 2, 96, 32, True, True, False, "fp16", "fp16"),
    (2, 5, 1, 256, 256, False, True, False, "fp32", "bf16"),
    (2, 3, 3, 250, 250, True, True, True, "fp16", "fp32"),   # no vector loads: odd pairs of channels
    (3, 2, 1, 18, 6, False, True, True, "bf16", "fp16"),
    (3, 2, 1, 2, 2, True, True, True, "fp32", "fp32"),
    (4, 2, 1, 64, 0, False, True, False, "bf16", "bf16"),    # nothing rotated
    (1030, 6, 2, 64, 32, True, True, True, "bf16", "fp16"),  # a block walks over a token's heads
])
def test_qk_norm_rope(tokens, nh, nkv, hd, rot, inter, norm, bias, tin, tout):
    rng = np.random.default_rng(tokens * hd + rot)
    n = (nh + 2 * nkv) * hd
    qkv, x = _rand(rng, (tokens, n), tin, 3.0)
    cos, sin = (A.rope_tables_scaled(rot, 1e6, 3000) if rot else (np.zeros((3000, 0), np.float32),) * 2)
    pos = rng.integers(0, 3000, tokens).astype(np.int32)
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    wq, wk = ((1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32) if norm else (None, None))
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = A.qk_norm_rope(qkv, nh, nkv, up(cos), up(sin), up(pos), bias=up(b), q_norm=up(wq), k_norm=up(wk), eps=1e-5,
                         interleaved=inter, out_dtype=DT[tout])
    ref = R.rope(x, nh, nkv, cos, sin, pos, b, wq, wk, 1e-5, inter)
    absolute = np.abs(x).max() + (np.abs(b).max() if bias else 0)
    for g, (y, size) in zip(got, ref):
        assert g.dtype == DT[tout]
        # fp32: the bias (on |x| + |b|, before any scaling), the norm's sum of hd squares (half of hd + its square
        # root, division and two products), two products and a sum; then the rounding to the type
        grow = np.abs(y).max() / absolute if norm else 1.0
        bound = E32 * ((6 + hd / 2) * size * 2 + 2 * absolute * max(grow, 1.0)) + R.HALF[tout] * np.abs(y) + 1e-30
        if tout == "fp16":
            bound = bound + 2.0 ** -25
        _close(g, y, bound)


def test_qk_norm_rope_padding_views_and_in_place():
    """Padding rows stay, strided rows and outputs that are views, rotation in the rows themselves, an odd alignment."""
    rng = np.random.default_rng(1)
    nh, nkv, hd = 4, 2, 64
    n = (nh + 2 * nkv) * hd
    cos, sin = A.rope_tables_scaled(hd, 1e4, 50)
    pos = torch.tensor([3, -1, 49, 50, 7], dtype=torch.int32, device="cuda")
    cos_d, sin_d = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    for shift in (0, 1):
        big, _ = _rand(rng, (5, n + 24), "fp32")
        rows = big[:, 8 + shift:8 + shift + n]
        before = big.clone()
        ref = R.rope(_np(rows), nh, nkv, cos, sin, np.array([3, 0, 49, 0, 7]))
        fresh = A.qk_norm_rope(rows, nh, nkv, cos_d, sin_d, pos)
        parts = rows.split((nh * hd, nkv * hd, nkv * hd), dim=1)
        views = tuple(p.unflatten(1, (-1, hd)) for p in parts)
        A.qk_norm_rope(rows, nh, nkv, cos_d, sin_d, pos, out=views)
        for f, w, (y, size) in zip(fresh, views, ref):
            keep = [0, 2, 4]
            _close(f[keep], y[keep], 8 * E32 * size[keep])
            assert torch.equal(f[keep], w[keep])
            assert not f[[1, 3]].any()
        assert torch.equal(big[[1, 3]], before[[1, 3]])
        assert torch.equal(big[:, :8 + shift], before[:, :8 + shift])
        assert torch.equal(big[:, 8 + shift + n:], before[:, 8 + shift + n:])


# ---- the cache --------------------------------------------------------------------------
def _caches(pages, page, nkv, hd, seed=9):
    raw = np.random.default_rng(seed).integers(0, 256, (pages, nkv, page // 16, 20 * hd), dtype=np.uint8)
    return torch.from_numpy(raw.copy()).cuda(), raw


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("tokens,nkv,hd,page,vec", [(1, 1, 64, 16, True), (9, 3, 128, 32, True), (50, 2, 64, 48, False),
                                                     (130, 4, 128, 16, False)])
def test_append_bits_and_read(dtype, tokens, nkv, hd, page, vec):
    """The cache's bytes are those of the definition, the rest of it stays, and it reads back as d * n + m."""
    rng = np.random.default_rng(tokens)
    pages = -(-2 * tokens // page) + 1
    cache, raw = _caches(pages, page, nkv, hd)
    pad = 0 if vec else 3
    k, kx = _rand(rng, (tokens, nkv, hd + pad), dtype, 2.0)
    v, vx = _rand(rng, (nkv, tokens, hd), dtype)
    k, kx = k[..., pad:], kx[..., pad:]      # an odd start: no vector loads
    v, vx = v.transpose(0, 1), vx.transpose(1, 0, 2)  # heads before tokens
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 8:
        slots[[2, 5, 7]] = [-1, pages * page, 1 << 60]
    ds = torch.from_numpy(slots).cuda()
    A.kv_append_q4(cache, k, v, ds)
    R.write(raw, kx.astype(np.float32), vx.astype(np.float32), slots)
    assert np.array_equal(cache.cpu().numpy(), raw)
    kk, vv, ks, vs = R.unpack(raw)
    live = (slots >= 0) & (slots < pages * page)
    for out in ("fp32", dtype):
        got = A.kv_read_q4(cache, ds, dtype=DT[out])
        for g, x, size in zip(got, (kk, vv), (ks, vs)):
            x, size = (y.transpose(0, 2, 1, 3).reshape(-1, nkv, hd)[np.where(live, slots, 0)] for y in (x, size))
            assert not g[torch.from_numpy(~live).cuda()].any()
            _close(g[torch.from_numpy(live).cuda()], x[live], (E32 * size + R.HALF[out] * np.abs(x) + 2.0 ** -25)[live])
    keep = torch.full((tokens, nkv, hd), 7.0, device="cuda")
    A.kv_read_q4(cache, torch.full_like(ds, -5), out=(keep, keep.clone()))
    assert bool((keep == 7).all())


def test_append_hard_values():
    """Ties between two nibbles, steps on the border of two fp16 values, groups that are constant, tiny, huge, beyond
    fp16's range, or not finite."""
    rng = np.random.default_rng(3)
    x = np.zeros((64, 1, 64), np.float32)
    for i in range(24):  # exact ties: m = 0, d = 2^(i - 12), x = (n + 1/2) d
        d = 2.0 ** (i - 12)
        x[i, 0, :32] = rng.integers(0, 15, 32) * d + d / 2
        x[i, 0, 0], x[i, 0, 1] = 0, 15 * d
        # steps halfway between two fp16 values, and an fp32 step to either side
        edge = np.float32(15 * d * (1 + (2 * rng.integers(0, 1023) + 1) * 2.0 ** -11))
        x[i, 0, 32:] = rng.random(32) * edge
        x[i, 0, 32], x[i, 0, 33] = 0, [edge, np.nextafter(edge, np.float32(0)), np.nextafter(edge, np.float32(9e9))][i % 3]
    x[24] = 1000.25
    x[25, 0, :32] = -3e38 + rng.random(32) * 6e38
    x[26, 0, :32] = 1e-7 * rng.standard_normal(32)
    x[27, 0, :32] = 1e-30 * rng.standard_normal(32)
    x[28, 0, :32] = 1e6 + rng.random(32)
    x[29, 0, :32] = -1e6 - rng.random(32)
    x[30, 0, :32] = 70000 * rng.random(32)
    x[31, 0, 5], x[32, 0, 37], x[33, 0, 63] = np.nan, np.inf, -np.inf
    x[34, 0, :32] = 65504 * (1 - 2 * rng.integers(0, 2, 32))
    x[35, 0, :32] = np.float32(6.1e-5) * 15 * rng.random(32)
    for i in range(36, 64):
        x[i] = rng.standard_normal((1, 64)) * 10.0 ** rng.integers(-8, 5)
    t = torch.from_numpy(x).cuda()
    cache, raw = _caches(4, 16, 1, 64)
    slots = np.arange(64)
    A.kv_append_q4(cache, t, -t, torch.from_numpy(slots).cuda())
    R.write(raw, x, -x, slots)
    assert np.array_equal(cache.cpu().numpy(), raw)
    k, v = A.kv_read_q4(cache, torch.from_numpy(slots).cuda())
    kk, vv, _, _ = R.unpack(raw)
    assert np.isnan(_np(k)[31, 0, :32]).all() and np.isnan(_np(v)[33, 0, 32:]).all()
    _close(k, kk.transpose(0, 2, 1, 3).reshape(64, 1, 64), E32 * 2 * np.abs(np.nan_to_num(x)).clip(max=1.1e6) + 1e-12)


# ---- decode attention ----------------------------------------------------------------------
def _decode_bound(q, k, ks, v, vs, scale, o, dtype):
    """How far a decode output may be off.

    Scores: sums of hd products of 16-bit pieces in fp32, each sum and scaling off by E32 of the sum of the parts'
    sizes |q| (|d n| + |m|); 40 such roundings at most (a product's own, adders of 16 terms hd / 16 and 32 / 16
    deep that may cut instead of round, the pieces of q, the scales), 1 for exp2's argument: delta; softmax
    weights are off by e^(2 delta) - 1.  The weights are applied to values in pieces: exact to E32 in fp32 (64
    roundings: running rescales, the split sums), to fp16 once and once with the step in the 16-bit types."""
    size = (np.abs(q)[:, None] * ks[None]).sum(-1) * scale
    s = (q @ k.T) * scale
    delta = 40 * E32 * size.max(-1) + 2 * E32 * np.abs(s).max(-1) + 4 * E32
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    step = 64 * E32 if dtype == "fp32" else 2 * 2.0 ** -11 + 64 * E32
    return ((np.expm1(2 * delta)[:, None] + step) * (p @ vs) + R.HALF[dtype] * np.abs(o) + 1e-9 * np.nanmax(vs) +
            (2.0 ** -25 if dtype == "fp16" else 0))


def _decode_case(seed, lens, nh, nkv, hd, page, dtype, extra_pages=2, std=1.0, q_std=1.0):
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra_pages
    cache, raw = _caches(pages, page, nkv, hd, seed)  # what is not written stays random bytes: NaN scales among them
    order = rng.permutation(pages)
    table = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    slots, ks, vs = [], [], []
    channel = np.where(np.arange(hd) % 17 == 3, 9.0, 1.0)
    for b, n in enumerate(lens):
        t = np.arange(n)
        slots.append(table[b, t // page].astype(np.int64) * page + t % page)
        ks.append((rng.standard_normal((n, nkv, hd)) * channel + 0.3 * channel).astype(np.float32))
        vs.append((rng.standard_normal((n, nkv, hd)) * std).astype(np.float32))
    cat = lambda a: torch.from_numpy(np.concatenate(a)).cuda()  # noqa: E731
    A.kv_append_q4(cache, cat(ks), cat(vs), cat(slots))
    q, qx = _rand(rng, (len(lens), nh, hd), dtype, q_std)
    return cache, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), q, qx


def _decode_ref(cache, table, lens, qx, scale, dtype, page, skewed=False):
    with np.errstate(all="ignore"):
        kk, vv, ks, vs = R.unpack(cache.cpu().numpy())
        if skewed:
            vs = np.maximum(vs, R.middle_sizes(cache.cpu().numpy()))
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    out, bound = np.zeros_like(qx), np.zeros_like(qx)
    group = qx.shape[1] // kk.shape[1]
    for b in range(len(lens)):
        t = np.arange(max(0, min(int(lens[b]), table.shape[1] * page)))
        pg = table[b, t // page]
        t = t[(pg >= 0) & (pg < kk.shape[0])]
        if not len(t):
            continue
        pg = table[b, t // page]
        for h in range(kk.shape[1]):
            k, v, k_size, v_size = (x[pg, h, t % page] for x in (kk, vv, ks, vs))
            rows = slice(h * group, (h + 1) * group)
            o, _ = R.attend(qx[b, rows], k, v, scale)
            out[b, rows], bound[b, rows] = o, _decode_bound(qx[b, rows], k, k_size, v, v_size, scale, o, dtype)
    return out, bound


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("lens,nh,nkv,hd,page", [
    ([1], 1, 1, 64, 16),
    ([0, 1, 15, 16, 17, 0], 8, 2, 128, 16),
    ([33, 250, 1], 28, 4, 128, 32),
    ([700], 28, 4, 128, 64),
    ([129, 64, 5], 14, 2, 64, 48),
    ([40, 300], 32, 2, 128, 16),   # 16 query heads a KV head
    ([90], 11, 1, 64, 16),          # 11: two parts of unequal heads
    ([3000, 1, 1, 900], 6, 2, 64, 16),
    ([20000], 2, 1, 64, 64),                       # cut into more than 32 pieces
    ([5, 0, 40] * 100 + [700], 3, 1, 64, 16),     # more sequences than threads of a CTA
])
def test_decode_q4(dtype, lens, nh, nkv, hd, page):
    cache, table, n, q, qx = _decode_case(len(lens) + nh, lens, nh, nkv, hd, page, dtype)
    got = A.attention_decode_q4(q, cache, table, n)
    ref, bound = _decode_ref(cache, table, n, qx, hd ** -0.5, dtype, page)
    _close(got, ref, bound)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_decode_q4_sizes_of_values(dtype):
    """Queries and values far from one: scores of hundreds (one token takes all), values of 1e-5 and 1e4, and all of
    them zero."""
    for q_std, std in ((30.0, 1.0), (1e-4, 1e-5), (1.0, 1e4), (1e-30, 1.0), (1.0, 0.0), (0.0, 1.0)):
        cache, table, n, q, qx = _decode_case(5, [100, 37], 8, 2, 128, 16, dtype, std=std, q_std=q_std)
        got = A.attention_decode_q4(q, cache, table, n, scale=0.2)
        ref, bound = _decode_ref(cache, table, n, qx, float(np.float32(0.2)), dtype, 16)
        _close(got, ref, bound + 1e-30)


def test_decode_q4_long_sums_keep_fp32():
    """Over tens of thousands of tokens fp32 results stay fp32: what roundings of either sign leave of 16 a term, 16 * E32
    of the result's norm.  (Sums that are cut towards zero, as the tensor cores' are, lose half a step each time: 1e-5
    over 60000 tokens if they ran through.)"""
    cache, table, n, q, qx = _decode_case(6, [60000], 4, 1, 64, 128, "fp32")
    got = _np(A.attention_decode_q4(q, cache, table, n))
    ref, _ = _decode_ref(cache, table, n, qx, 0.125, "fp32", 128)
    assert np.linalg.norm(got - ref) <= 16 * E32 * np.linalg.norm(ref)


def test_decode_q4_bad_tables_lengths_and_strides():
    """Page numbers outside the cache hide their tokens, lengths are held to the table, strided queries and outputs,
    and what lies beside the output stays."""
    cache, table, n, q, qx = _decode_case(7, [100, 70, 64, 48], 8, 2, 64, 16, "fp32")
    table[0, 2], table[1, 0], table[1, 4] = 1 << 30, -7, cache.shape[0]
    table[2] = -1
    n[3] = 1 << 30
    table[3, 3:] = table[0, 0]
    wide = torch.full((4, 9, 80), 5.0, device="cuda")
    out = wide[:, :8, 8:72]
    strided = torch.zeros(8, 4, 64, device="cuda").transpose(0, 1)
    strided.copy_(q)
    got = A.attention_decode_q4(strided, cache, table, n, out=out)
    assert got is out
    ref, bound = _decode_ref(cache, table, n, qx, 0.125, "fp32", 16)
    _close(out, ref, bound)
    assert not out[2].any()
    assert bool((wide[:, 8] == 5).all() and (wide[:, :, :8] == 5).all() and (wide[:, :, 72:] == 5).all())
    # queries and outputs that allow no vector access
    odd = torch.full((4, 8 * 65 + 1), 3.0, device="cuda")
    q_odd, o_odd = (t[:, 1:].view(4, 8, 65)[..., :64] for t in (odd.clone(), odd))
    q_odd.copy_(q)
    A.attention_decode_q4(q_odd, cache, table, n, out=o_odd)
    assert torch.equal(o_odd, out) and bool((odd[:, 0] == 3).all())
    n.fill_(-3)
    assert not A.attention_decode_q4(q, cache, table, n).any()
    assert A.attention_decode_q4(q, cache, table[:, :0], n.fill_(9)).abs().sum() == 0
    assert A.attention_decode_q4(q[:0], cache, table[:0], n[:0]).shape == (0, 8, 64)


def test_decode_q4_not_finite():
    """A cached group that is not finite: NaN in V reaches its 32 channels, NaN in K the heads that read it."""
    cache, table, n, q, qx = _decode_case(8, [40, 40], 4, 2, 64, 16, "fp32")
    bad = torch.ones(2, 2, 64, device="cuda")
    bad[0, 0, 40] = float("nan")   # slot of sequence 0, head 0
    ones = torch.ones(2, 2, 64, device="cuda")
    at = [int(table[b, 1]) * 16 + 3 for b in (0, 1)]
    A.kv_append_q4(cache, ones, bad, torch.tensor(at).cuda())
    A.kv_append_q4(cache, bad.flip(0), ones, torch.tensor([at[0] + 1, at[1] + 1]).cuda())
    got = A.attention_decode_q4(q, cache, table, n)
    ref, bound = _decode_ref(cache, table, n, qx, 0.125, "fp32", 16)
    assert np.isnan(ref[0, :2, 32:]).all() and np.isfinite(ref[0, :2, :32]).all() and np.isnan(ref[1, :2]).all()
    assert np.isfinite(ref[:, 2:]).all()
    _close(got, ref, bound)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_decode_q4_values_beyond_fp16(dtype):
    """Groups whose middle m + 8 d lies above 65504, in whole blocks and in a sequence's last one (in fp16 few and with
    small weights, so that the results stay inside the type).  Weights are applied to n - 8 and m + 8 d, so in a
    group that lies to one side of its offset their roundings count by |d (n - 8)| + |m + 8 d|, which at n = 0 is more
    than |m| = |d n| + |m|."""
    cache, table, n, q, qx = _decode_case(9, [100, 37, 64], 8, 2, 128, 16, dtype)
    rng = np.random.default_rng(10)
    at = [(0, 20), (0, 99), (1, 5), (1, 36), (2, 63)]
    slots = torch.tensor([int(table[b, t // 16]) * 16 + t % 16 for b, t in at]).cuda()
    k, v = (np.asarray(rng.standard_normal((5, 2, 128)) * s, np.float32) for s in (1.0, 2e5))
    if dtype == "fp16":
        v *= 1e-2
        v[:, 0, 40:72] = 6e4
        v[:, 0, 50] = 4e5
    A.kv_append_q4(cache, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slots)
    got = A.attention_decode_q4(q, cache, table, n, scale=0.01)
    ref, bound = _decode_ref(cache, table, n, qx, float(np.float32(0.01)), dtype, 16, skewed=True)
    assert np.abs(ref).max() < 65000
    _close(got, ref, bound)


@pytest.mark.parametrize("std", [1e-5, 1e-3, 1e-2, 1.0, 1e3, 1e4, 1e5])
def test_decode_q4_fp32_at_any_size_of_values(std):
    """Equal weights (queries of zero), so that only the values' way counts.  Weights times steps and offsets m + 8 d are
    in two halves each: 2^-22, 4 * E32; the rest of an offset's weight another 4 * E32; four sums of 16 terms that may
    cut, 8 * E32; sums over blocks and warps and the division, 8 * E32: 24 * E32 of the terms' sizes."""
    cache, table, n, q, qx = _decode_case(12, [90, 17], 4, 2, 128, 16, "fp32", std=std, q_std=0.0)
    with np.errstate(all="ignore"):
        _, vv, _, vs = R.unpack(cache.cpu().numpy())
    got = _np(A.attention_decode_q4(q, cache, table, n))
    for b, tokens in enumerate(n.tolist()):
        t = np.arange(tokens)
        pg = table[b].cpu().numpy()[t // 16]
        for h in range(2):
            v, size = vv[pg, h, t % 16], vs[pg, h, t % 16]
            assert np.all(np.abs(got[b, 2 * h:2 * h + 2] - v.mean(0)) <= 24 * E32 * size.mean(0))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_decode_q4_queries_not_finite(dtype):
    """An infinity or a NaN in a query makes its head's results NaN, as it makes every score, and no other's."""
    cache, table, n, q, qx = _decode_case(13, [40, 3, 0], 4, 2, 64, 16, dtype)
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = q.clone()
        x[:, 1, 7] = bad
        got = A.attention_decode_q4(x, cache, table, n)
        ref, bound = _decode_ref(cache, table, n, qx, 0.125, dtype, 16)
        assert bool(torch.isnan(got[:2, 1]).all()) and not got[2].any()
        _close(got[:, [0, 2, 3]], ref[:, [0, 2, 3]], bound[:, [0, 2, 3]])


# ---- prompt attention ------------------------------------------------------------------------
def _prefill_ref(qx, kx, vx, cu_q, cu_k, causal, scale, dtype):
    nh, nkv = qx.shape[1], kx.shape[1]
    out, bound = np.zeros_like(qx), np.zeros_like(qx)
    for b in range(len(cu_q) - 1):
        (q0, q1), (k0, k1) = cu_q[b:b + 2], cu_k[b:b + 2]
        nq, nk = q1 - q0, k1 - k0
        seen = np.ones((nq, nk), bool)
        if causal:
            seen = np.arange(nk)[None] <= np.arange(nq)[:, None] + nk - nq
        for h in range(nh):
            q, k, v = qx[q0:q1, h], kx[k0:k1, h * nkv // nh], vx[k0:k1, h * nkv // nh]
            with np.errstate(all="ignore"):
                o, p_abs = R.attend(q, k, v, scale, seen)
                # scores: hd products summed in fp32 (16 at a time, cut or rounded) and scaled: hd + 8 roundings
                # of the sizes; weights rounded once to the type, their sum (64 + nk / 16 roundings in fp32) is not
                size = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0.0).max(-1, initial=0.0)
                delta = (qx.shape[2] + 8) * E32 * size
                step = R.HALF[dtype] + (64 + nk / 16) * E32 + np.expm1(2 * delta)
                out[q0:q1, h] = o
                bound[q0:q1, h] = step[:, None] * p_abs + R.HALF[dtype] * np.abs(o) + 2.0 ** -25
    return out, bound


def _prefill_case(seed, qs, ks, nh, nkv, hd, dtype, pad=0, std=1.0):
    rng = np.random.default_rng(seed)
    q, qx = _rand(rng, (sum(qs) + pad, nh, hd), dtype, std)
    k, kx = _rand(rng, (sum(ks) + pad, nkv, hd), dtype)
    v, vx = _rand(rng, (sum(ks) + pad, nkv, hd), dtype)
    cu = [np.concatenate([[0], np.cumsum(x)]).astype(np.int32) for x in (qs, ks)]
    return q, k, v, *(torch.from_numpy(c).cuda() for c in cu), (qx, kx, vx, *cu)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qs,ks,nh,nkv,hd", [
    ([1], [1], 1, 1, 64),
    ([77], [77], 4, 2, 128),
    ([128], [128], 2, 1, 64),
    ([129, 1, 255], [129, 1, 255], 4, 2, 64),
    ([256, 257], [256, 257], 3, 3, 128),
    ([5, 0, 300, 64], [400, 7, 300, 64], 8, 2, 128),     # tokens before the prompt; a sequence without queries
    ([200, 30], [60, 0], 2, 2, 64),                       # more queries than keys: rows that see nothing
    ([700], [900], 6, 1, 128),
    ([1, 1, 1, 2, 1, 3] * 9, [4, 1, 9, 2, 130, 3] * 9, 2, 1, 64),
    ([100, 37], [100, 50], 14, 2, 64),                     # seven heads a tile, 126 rows of it
    ([40], [40], 11, 1, 128),                              # eleven: one a tile
    ([9, 3], [9, 300], 96, 1, 64),                         # 96 = 32 * 3: 32 heads a tile
])
def test_prefill(dtype, causal, qs, ks, nh, nkv, hd):
    q, k, v, cu_q, cu_k, x = _prefill_case(len(qs) + hd + nh, qs, ks, nh, nkv, hd, dtype, pad=3)
    out = torch.full_like(q, 3.0)
    got = A.attention_prefill(q, k, v, cu_q, cu_k, causal=causal, out=out)
    assert got is out
    n = sum(qs)
    ref, bound = _prefill_ref(*x, causal, hd ** -0.5, dtype)
    _close(out[:n], ref[:n], bound[:n])
    assert bool((out[n:] == 3).all())


def test_prefill_strides_scale_and_defaults():
    """Views of one projection, heads before tokens, a scale, cu_k left out, large scores."""
    rng = np.random.default_rng(11)
    nh, nkv, hd, t = 4, 2, 64, 150
    qkv, _ = _rand(rng, (t, (nh + 2 * nkv) * hd), "bf16", 3.0)
    q, k, v = (p.unflatten(1, (-1, hd)) for p in qkv.split((nh * hd, nkv * hd, nkv * hd), dim=1))
    cu = torch.tensor([0, 50, 150], dtype=torch.int32).cuda()
    out = torch.full((nh, t, hd), 2.0, dtype=torch.bfloat16, device="cuda")
    A.attention_prefill(q, k, v, cu, scale=0.5, out=out.transpose(0, 1))
    ref, bound = _prefill_ref(_np(q), _np(k), _np(v), [0, 50, 150], [0, 50, 150], True, 0.5, "bf16")
    _close(out.transpose(0, 1), ref, bound)
    again = A.attention_prefill(q.contiguous(), k.transpose(0, 1).contiguous().transpose(0, 1), v, cu, scale=0.5)
    assert torch.equal(again, out.transpose(0, 1))
    for scale in (0.0, -0.3):
        got = A.attention_prefill(q, k, v, cu, scale=scale)
        ref, bound = _prefill_ref(_np(q), _np(k), _np(v), [0, 50, 150], [0, 50, 150], True, scale, "bf16")
        _close(got, ref, bound)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prefill_hidden_values_have_no_part(dtype):
    """NaN and infinities where no query looks: rows of no sequence, the next sequence, and later keys of the own one."""
    q, k, v, cu_q, cu_k, x = _prefill_case(3, [150, 70], [150, 70], 2, 1, 64, dtype, pad=40)
    qx, kx, vx, *cu = x
    for t, a in ((k, kx), (v, vx)):
        t[220:], a[220:] = float("nan"), np.nan
        t[219], a[219] = float("inf"), np.inf     # the second sequence's last key: only its last query sees it
        t[100], a[100] = float("nan"), np.nan     # the first sequence's queries from 100 on see it
    q[220:] = float("nan")
    got = A.attention_prefill(q, k, v, cu_q, cu_k)
    ref, bound = _prefill_ref(qx, kx, vx, *cu, True, 0.125, dtype)
    seen = [*range(100), *range(150, 219)]
    _close(got[seen], ref[seen], bound[seen])
    assert bool(torch.isnan(got[100:150]).all()) and bool(torch.isnan(got[219]).all())
    assert not got[220:].any()


def test_prefill_scores_of_minus_infinity():
    """A key of score -inf has no weight, and a query that sees no other gets 0 / 0."""
    q, k, v, cu_q, cu_k, x = _prefill_case(7, [140], [140], 2, 1, 64, "bf16")
    qx, kx, vx, *cu = x
    q[..., 3], qx[..., 3] = 1.0, 1.0
    k[0, 0, 3], kx[0, 0, 3] = float("-inf"), -np.inf
    got = A.attention_prefill(q, k, v, cu_q, cu_k)
    kx[0] = 0.0  # (for the reference: the key is left out)
    for h in range(2):
        seen = np.tril(np.ones((140, 140), bool))
        seen[:, 0] = False
        ref, p_abs = R.attend(qx[:, h], kx[:, 0], vx[:, 0], 0.125, seen)
        size = (np.abs(qx[:, h]) @ np.abs(kx[:, 0]).T * 0.125).max(-1)
        step = R.HALF["bf16"] + 73 * E32 + np.expm1(2 * 72 * E32 * size)
        _close(got[1:, h], ref[1:], step[1:, None] * p_abs[1:] + R.HALF["bf16"] * np.abs(ref[1:]) + 2.0 ** -25)
    assert bool(torch.isnan(got[0]).all())


def test_no_tokens():
    """Calls without a token launch nothing and return what has the right shape."""
    z = lambda *s, d=torch.float32: torch.zeros(*s, dtype=d, device="cuda")  # noqa: E731
    q, k, v = A.qk_norm_rope(z(0, 8 * 64), 4, 2, z(5, 32), z(5, 32), z(0, d=torch.int32))
    assert q.shape == (0, 4, 64) and k.shape == v.shape == (0, 2, 64)
    cache, slots = A.kv_cache_q4(1, 16, 2, 64), z(0, d=torch.int64)
    A.kv_append_q4(cache, k, v, slots)
    assert not cache.any() and A.kv_read_q4(cache, slots)[0].shape == (0, 2, 64)
    h = torch.float16
    out = A.attention_prefill(z(0, 4, 64, d=h), z(3, 2, 64, d=h), z(3, 2, 64, d=h), z(2, d=torch.int32))
    assert out.shape == (0, 4, 64)
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    out = A.attention_prefill(z(2, 4, 64, d=h) + 1, z(0, 2, 64, d=h), z(0, 2, 64, d=h), cu, z(2, d=torch.int32))
    assert not out.any()


def test_bad_ends_stay_inside():
    """Ends that fall, or lie outside the rows, are held to them: nothing outside is touched."""
    q, k, v, _, _, _ = _prefill_case(4, [64], [64], 2, 1, 64, "bf16")
    for ends in ([5, 3, 70], [-9, 1 << 30, 2], [64, 0, 0]):
        cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
        guard = torch.full((68, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        A.attention_prefill(q, k, v, cu, out=guard[2:66])
        torch.cuda.synchronize()
        assert bool((guard[:2] == 7).all() and (guard[66:] == 7).all())


def test_first_calls_inside_a_capture():
    """In a fresh process: every operator's first call is captured, and the replay gives what an eager call gives."""
    import subprocess
    import sys

    code = """
import torch
from flatrun_b200 import attention as A
z = lambda *s, d=torch.float32: torch.randn(*s, device="cuda").to(d)
qkv, pos = z(3, 8 * 64), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
cos, sin = (torch.from_numpy(t).cuda() for t in A.rope_tables_scaled(64, 1e4, 9))
cache, slots = A.kv_cache_q4(1, 16, 2, 64), torch.arange(3, device="cuda")
table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
n, cu = torch.tensor([3], dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
def step():
    q, k, v = A.qk_norm_rope(qkv, 4, 2, cos, sin, pos, out_dtype=torch.float16)
    A.kv_append_q4(cache, k, v, slots)
    return A.attention_prefill(q, k, v, cu), A.attention_decode_q4(q[2:], cache, table, n), A.kv_read_q4(cache, slots)[0]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step())) and all(bool(t.any()) for t in got)
print("captured")
"""
    import os
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=repo, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---- as they are used together ---------------------------------------------------------------
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 64)])
def test_prompt_then_decode(hd, page):
    """Prompts of three sequences, then tokens one by one: rotation, prompt attention, the cache, decode attention,
    eagerly on a stream of its own, then the token step captured and replayed with new positions."""
    rng = np.random.default_rng(21)
    nh, nkv = 8, 2
    n = (nh + 2 * nkv) * hd
    lens = [50, 1, 131]
    cos, sin = A.rope_tables_scaled(hd, 1e6, 400)
    pages = 16 * 64 // page
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cos_d, sin_d = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        cache = A.kv_cache_q4(pages, page, nkv, hd)
        table = torch.from_numpy(rng.permutation(pages)[:3 * (pages // 3)].reshape(3, -1).astype(np.int32)).cuda()
        rows, x = _rand(rng, (sum(lens), n), "fp32", 1.5)
        pos = np.concatenate([np.arange(m) for m in lens]).astype(np.int32)
        seq = np.repeat(np.arange(3), lens)
        th = table.cpu().numpy()
        slots = th[seq, pos // page].astype(np.int64) * page + pos % page
        q, k, v = A.qk_norm_rope(rows, nh, nkv, cos_d, sin_d, torch.from_numpy(pos).cuda(), out_dtype=torch.bfloat16)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
        o = A.attention_prefill(q, k, v, cu)
        A.kv_append_q4(cache, k, v, torch.from_numpy(slots).cuda())
        ref, bound = _prefill_ref(_np(q), _np(k), _np(v), cu.tolist(), cu.tolist(), True, hd ** -0.5, "bf16")
        _close(o, ref, bound)

        new, _ = _rand(rng, (3, n), "fp32", 1.5)
        position = torch.tensor(lens, dtype=torch.int32).cuda()
        out = torch.zeros((3, nh, hd), device="cuda")
        tok = tuple(torch.zeros((3, h, hd), device="cuda") for h in (nh, nkv, nkv))
        which = torch.arange(3, device="cuda")

        def step():
            A.qk_norm_rope(new, nh, nkv, cos_d, sin_d, position, out=tok)
            slot = table[which, (position // page).long()].long() * page + position % page
            A.kv_append_q4(cache, tok[1], tok[2], slot)
            position.add_(1)
            A.attention_decode_q4(tok[0], cache, table, position, out=out)

        def check():
            stream.synchronize()
            ref, bound = _decode_ref(cache, table, position, _np(tok[0]), hd ** -0.5, "fp32", page)
            _close(out, ref, bound)

        step()
        check()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(3):
            new.copy_(torch.from_numpy(rng.standard_normal((3, n)).astype(np.float32)))
            graph.replay()
            check()
        assert position.tolist() == [m + 4 for m in lens]


def test_calls_on_two_streams_at_once():
    """Two decode calls in flight on two streams give what each gives alone."""
    a = _decode_case(31, [2000, 900, 1], 8, 2, 128, 16, "bf16")
    b = _decode_case(32, [1, 3000], 8, 2, 128, 16, "bf16")
    alone = [A.attention_decode_q4(c[3], c[0], c[1], c[2]) for c in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, c in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(A.attention_decode_q4(c[3], c[0], c[1], c[2]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g, alone[i]) for g in got[i])


# ---- the decode engine's paths ---------------------------------------------------------------
def _engine(**kw):
    import qwen2_restated as Q
    from flatrun_b200.decode import DecodeEngine, DecoderConfig

    s = Q.TINY
    scaling = kw.pop("rope_scaling", None)
    cfg = DecoderConfig(s.H, s.F, s.V, s.L, s.NH, s.NKV, s.EPS, s.THETA, 100, scaling)
    return DecodeEngine(cfg, Q.build(s), lambda name: Q.quant_of(s, name), **kw)


def _run(eng, tokens):
    out = []
    for t in tokens:
        eng.step(int(t))
        out.append(eng.logits_host())
    return np.stack(out)


def test_engine_with_a_4_bit_cache():
    """The 4-bit engine runs eagerly and captured with the same logits, and its first layer's cache holds what the
    fp32 engine's does, to half a step."""
    tokens = np.random.default_rng(5).integers(0, 320, 40)
    full = _engine()
    _run(full, tokens)
    eager, graph = _engine(kv_bits=4, kv_page=16), _engine(kv_bits=4, kv_page=16)
    graph.capture()
    got = _run(eager, tokens)
    assert np.array_equal(got, _run(graph, tokens))
    assert np.isfinite(got).all() and int(graph.pos.item()) == 40 and int(graph._slot.item()) == 40
    k, v = A.kv_read_q4(eager.q4_cache[0], torch.arange(40, device="cuda"))
    for x, y in ((full.k_cache[0][:40], k), (full.v_cache[0][:40], v)):
        x = _np(x)
        _, d, _ = R.quantise(x)
        # half a step, the roundings of d and m to fp16 (as in the round trip of the oracle), and the engines' own
        # differences before the cache (rotation in fp32: 8 roundings)
        bound = np.repeat(d, 32, -1) * (0.5 + 15 * 2.0 ** -11) + np.abs(x).max() * (2.0 ** -11 + 16 * E32)
        _close(y, x, bound)
    # the last layer's attention of the last token, from the queries and the cache that the engine holds
    q = eager.qkv[:eager.cfg.hidden].view(1, -1, 64)
    o, bound = _decode_ref(eager.q4_cache[-1], eager._table, torch.tensor([40]), _np(q), 0.125, "fp32", 16)
    _close(eager.ctx.view(1, -1, 64), o, bound)


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("parts", [(33,), (1, 5), (20, 17)])
def test_engine_prefill(bits, parts):
    """A prompt at once (and a second one behind it), then single tokens, against the same tokens one by one.

    The first layer's keys and values differ by the fp16 roundings of the batched projection's operands: 2 * 2^-11 of the
    sum of |x w| over 256 products, which is below three times the largest key (for products of one size with random
    signs it is 0.8 * 16 times the spread of the keys), and in 4 bits by a step more (a rounding can fall the other way).
    Later layers of this random model have scores of thousands, where a near tie between two keys can go either way
    anywhere, so beyond the first layer only the last token's logits are compared, loosely."""
    rng = np.random.default_rng(sum(parts))
    prompts = [rng.integers(0, 320, n) for n in parts]
    one, eng = _engine(kv_bits=bits), _engine(kv_bits=bits)
    for t in np.concatenate(prompts):
        one.step(int(t))
    ref = one.logits_host().copy()
    for p in prompts:
        eng.prefill(p)
    n = sum(parts)
    got = eng.logits_host().copy()
    assert eng.argmax_host() == int(np.argmax(got)) and int(eng.pos.item()) == n
    if bits == 32:
        pairs = [(c[0][:n], d[0][:n]) for c, d in ((one.k_cache, eng.k_cache), (one.v_cache, eng.v_cache))]
        assert np.abs(got - ref).max() <= 2e-2 * np.abs(ref).max()
    else:
        slots = torch.arange(n, device="cuda")
        pairs = zip(A.kv_read_q4(one.q4_cache[0], slots), A.kv_read_q4(eng.q4_cache[0], slots))
    for x, y in pairs:
        x = _np(x)
        _, d, _ = R.quantise(x)
        step = 0 if bits == 32 else np.repeat(d, 32, -1) * (1 + 2.0 ** -10 * 15)
        _close(y, x, 2 * 2.0 ** -11 * 3 * np.abs(x).max() + step)
    tail = _run(eng, rng.integers(0, 320, 3))
    assert np.isfinite(tail).all() and int(eng.pos.item()) == n + 3


def test_engine_options_and_refusals():
    with pytest.raises(ValueError, match="kv_bits"):
        _engine(kv_bits=8)
    eng = _engine(rope_scaling={"type": "linear", "factor": 2.0})
    with pytest.raises(ValueError, match="empty"):
        eng.prefill([])
    with pytest.raises(ValueError, match="max_pos"):
        eng.prefill(np.zeros(101, np.int32))
    for bad in (-1, 320):
        with pytest.raises(ValueError, match="token ids"):
            eng.prefill([3, bad])
    eng.step(3)
    eng.step(5)
    plain = _engine()
    plain.step(3)
    plain.step(5)
    eng.logits_host(), plain.logits_host()  # (waits for the engines' streams)
    assert torch.equal(eng.k_cache[0][0], plain.k_cache[0][0]) and not torch.equal(eng.k_cache[0][1], plain.k_cache[0][1])


def test_no_wait_ran_out():
    """The status word that bounded waits report to is clear after the calls above."""
    import ctypes

    from flatrun_b200 import _lib

    flags = ctypes.c_uint32(1)
    _lib.check(_lib.load().frc_device_status(0, ctypes.byref(flags)))
    assert flags.value == 0
