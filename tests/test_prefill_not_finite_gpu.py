"""Prompt attention with keys and values that are not finite (GPU): who sees them gets them, nobody else notices."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from flatrun_b200 import _lib, attention as A
import q4_restated as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
E32 = 2.0 ** -24


def _status():
    flags = ctypes.c_uint32(1)
    _lib.check(_lib.load().frc_device_status(0, ctypes.byref(flags)))
    return flags.value


def _case(seed, qs, ks, nh, nkv, hd, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q, k, v = (torch.randn((sum(n), h, hd), generator=g, device="cuda").to(DT[dtype])
               for n, h in ((qs, nh), (ks, nkv), (ks, nkv)))
    cu = [torch.tensor(np.concatenate([[0], np.cumsum(x)]), dtype=torch.int32, device="cuda") for x in (qs, ks)]
    return q, k, v, *cu


def _sees(qs, ks, causal):
    """(rows, keys): whether a row sees a key."""
    out = torch.zeros((sum(qs), sum(ks)), dtype=torch.bool)
    q0 = k0 = 0
    for nq, nk in zip(qs, ks):
        block = torch.ones((nq, nk), dtype=torch.bool)
        out[q0:q0 + nq, k0:k0 + nk] = block.tril(nk - nq) if causal else block
        q0, k0 = q0 + nq, k0 + nk
    return out.cuda()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qs,ks,nh,nkv,hd", [
    ([700], [700], 4, 2, 128),
    ([700], [700], 2, 2, 64),              # a head a tile: 256 queries an item, up to four tiles with masks
    ([300, 1, 513], [900, 1, 600], 8, 2, 64),
    ([130, 260], [130, 100], 4, 1, 128),   # rows that see nothing
    ([40] * 40, [140] * 40, 6, 2, 64),
])
def test_single_values_that_are_not_finite(dtype, causal, qs, ks, nh, nkv, hd):
    """V with single elements that are not finite against V with zeros in their places: rows that see one differ in its
    channel alone, where they are not finite; all else is equal bit for bit."""
    q, k, v, cu_q, cu_k = _case(len(qs) + hd, qs, ks, nh, nkv, hd, dtype)
    rng = np.random.default_rng(hd)
    n = sum(ks)
    bad = [(int(t), int(rng.integers(nkv)), int(rng.integers(hd))) for t in
           {0, 5, 127 % n, 128 % n, n // 2, n - 1, *rng.integers(0, n, 4)}]
    zeroed = v.clone()
    for i, at in enumerate(bad):
        v[at], zeroed[at] = [float("nan"), float("inf"), float("-inf")][i % 3], 0.0
    got, clean = (A.attention_prefill(q, k, x, cu_q, cu_k, causal=causal) for x in (v, zeroed))
    assert bool(torch.isfinite(clean).all())
    sees, hit = _sees(qs, ks, causal), torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    for t, h, c in bad:
        hit[:, h * nh // nkv:(h + 1) * nh // nkv, c] |= sees[:, t][:, None]
    assert not bool(torch.isfinite(got[hit]).any())
    assert torch.equal(got[~hit], clean[~hit])
    # an infinity alone in its channel, with weight, is what the sum is
    t, h, c = bad[1]
    if sum(b[1:] == (h, c) for b in bad) == 1:
        rows = got[:, h * nh // nkv, c][sees[:, t]]
        assert not bool((rows == float("-inf")).any())
    assert _status() == 0


def test_an_early_value_in_a_long_prompt():
    """A NaN in the first key's values: 5000 rows see it, and the call takes no multiple of its time (no row is
    computed a second time)."""
    q, k, v, cu_q, cu_k = _case(3, [5000], [5000], 8, 2, 128, "bf16")
    bad = v.clone()
    bad[0, 1, 77] = float("nan")

    def once(x):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        out = A.attention_prefill(q, k, x, cu_q, cu_k)
        b.record()
        b.synchronize()
        return a.elapsed_time(b), out

    once(v)
    (t_clean, clean), (t_bad, got) = (min((once(x) for _ in range(5)), key=lambda r: r[0]) for x in (v, bad))
    assert bool(torch.isnan(got[:, 4:, 77]).all())
    got[:, 4:, 77] = clean[:, 4:, 77] = 0
    # the first key's channel is the one that differs: NaN there, all else as without it
    assert torch.equal(got, clean)
    assert t_bad <= 3 * t_clean + 0.5
    assert _status() == 0


def test_other_sequences_behind_a_very_long_one():
    """300000 keys whose first is NaN in one channel, also hidden ones among the last: the sequences beside it get their
    results, and no wait runs out."""
    hd, n = 64, 300000
    qs, ks = [90, 300, 1], [n, 300, 77]
    q, k, v, cu_q, cu_k = _case(4, qs, ks, 2, 1, hd, "bf16")
    bad = v.clone()
    bad[0, 0, 9] = float("nan")
    bad[n - 40:n, 0, 20] = float("inf")  # the last 40 keys: only the last 40 queries see any
    got, clean = (A.attention_prefill(q, k, x, cu_q, cu_k) for x in (bad, v))
    assert bool(torch.isnan(got[:90, :, 9]).all())
    assert bool(torch.isfinite(got[:50, :, 20]).all()) and bool((got[50:90, :, 20] == float("inf")).all())
    assert torch.equal(got[90:], clean[90:]) and bool(torch.isfinite(got[90:]).all())
    assert _status() == 0
    # the rows themselves, where nothing is amiss: against 64 bits.  Scores: hd + 8 roundings of the sizes; the weights
    # rounded once to the type and their sum in fp32 (64 + n / 16 roundings)
    kx, vx = k[:n, 0].double().cpu().numpy(), v[:n, 0].double().cpu().numpy()
    for row in (0, 49):
        m = n - 89 + row
        for h in range(2):
            x = q[row, h].double().cpu().numpy()[None]
            o, p_abs = R.attend(x, kx[:m], vx[:m], 0.125)
            size = (np.abs(x) @ np.abs(kx[:m]).T * 0.125).max()
            step = R.HALF["bf16"] + (64 + m / 16) * E32 + np.expm1(2 * (hd + 8) * E32 * size)
            bound = step * p_abs + R.HALF["bf16"] * np.abs(o)
            keep = [c for c in range(hd) if c not in (9, 20)]
            assert np.all(np.abs(got[row, h].double().cpu().numpy() - o[0])[keep] <= bound[0][keep])
