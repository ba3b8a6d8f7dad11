"""What the decode engine decides on the host, on a stand-in without a GPU."""

from __future__ import annotations

import pytest
import torch

from flatrun_b200.decode import DecodeEngine, DecoderConfig


def _stand_in(max_pos: int, filled: int):
    """An engine of which only the position exists; its tokens are counted in `launched`."""
    eng = object.__new__(DecodeEngine)
    eng.torch, eng.lib, eng.stream, eng.kv_bits, eng._graph = torch, None, None, 32, None
    eng.cfg = DecoderConfig(64, 64, 16, 1, 1, 1, 1e-6, 1e4, max_pos)
    eng.pos, eng.tok_in = torch.tensor([filled]), torch.zeros(1, dtype=torch.int32)
    eng._filled = filled
    eng.launched = 0

    def token():
        eng.launched += 1

    eng._token = token
    return eng


def test_no_token_behind_max_pos():
    """The rotation's tables and the caches end at max_pos: a token there is refused before anything is launched."""
    eng = _stand_in(max_pos=5, filled=3)
    eng.step(1)
    eng.step()
    assert eng.launched == 2
    for call in (eng.step, eng.capture, lambda: eng.prefill([1])):
        with pytest.raises(ValueError, match="max_pos"):
            call()
    assert eng.launched == 2
    with pytest.raises(ValueError, match="max_pos"):
        _stand_in(max_pos=5, filled=3).prefill([1, 2, 3])


@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0), (3e4, 3e4, 6.5e4), (1.0, 1e6, 1.0), (1e5, 2.0, 3e9), (4e-3, 7e5, 1e-6),
                                   (1e5, 1e5, 1.0), (1e9, 1e9, 1e30), (2e4, 1e6, 0.0)])
@pytest.mark.parametrize("past", [0, 3])
def test_half_operands(sizes, past):
    """Nothing finite becomes infinite; scores and values are those of the fp32 operands to fp16's rounding of their
    sizes (three of 2^-11: two operands and their product's), except that scores come down by a power of two where
    queries and keys are both beyond 2^15; operands that fp16 holds are converted as they are."""
    from flatrun_b200.decode import _half_operands

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(5 + n, 2, 8, generator=g).clamp(-3, 3) / 3 * s for s, n in zip(sizes, (0, past, past)))
    k, v = ([x[:past], x[past:]] if past else [x] for x in (k, v))
    hq, hk, hv, up = _half_operands(q, k, v)
    k, v = torch.cat(k), torch.cat(v)
    assert all(x.dtype == torch.float16 and bool(torch.isfinite(x).all()) for x in (hq, hk, hv))
    assert hk.shape == k.shape and hv.shape == v.shape
    got, ref = (torch.einsum("thc,shc->tsh", x.double(), y.double()) for x, y in ((hq, hk), (q, k)))
    size = torch.einsum("thc,shc->tsh", q.double().abs(), k.double().abs())
    if max(sizes[0], sizes[1]) / 32768 * min(sizes[0], sizes[1]) > 32768:
        down = (ref / got).median().log2().round().exp2()
        assert down > 1
        got = got * down
    # (below 2^-14 fp16's steps are 2^-24: relative to the largest, at least 2^-24 / 2^-14)
    assert bool(((got - ref).abs() <= 3 * 2.0 ** -11 * size + 2.0 ** -10 * size.max() * 2.0 ** -10).all())
    assert bool(((hv.double() * up.double() - v.double()).abs() <= 2.0 ** -11 * v.double().abs() +
                 2.0 ** -25 * max(1.0, up)).all())
    if max(sizes) < 32768:
        assert up == 1 and torch.equal(hq, q.half()) and torch.equal(hk, k.half()) and torch.equal(hv, v.half())


def test_half_operands_not_finite():
    """An infinity or a NaN stays one, and changes nothing beside it."""
    from flatrun_b200.decode import _half_operands

    for bad in (float("inf"), float("nan")):
        q, k, v = (torch.ones(4, 1, 8) for _ in range(3))
        v[1, 0, 3] = bad
        hq, hk, hv, up = _half_operands(q, [k], [v])
        assert up == 1 and torch.equal(hq, q.half()) and torch.equal(hk, k.half())
        assert torch.equal(hv.isfinite(), v.isfinite()) and bool((hv[v.isfinite()] == 1).all())


def test_prefill_refuses_a_head_dim_before_anything_is_written():
    eng = _stand_in(max_pos=5, filled=0)
    eng.cfg = DecoderConfig(80, 64, 16, 1, 1, 1, 1e-6, 1e4, 5)
    with pytest.raises(ValueError, match="head_dim"):
        eng.prefill([1, 2])


def test_step_refuses_tokens_that_the_vocabulary_does_not_have():
    """The embedding's row is read without a check on the device."""
    eng = _stand_in(max_pos=9, filled=0)  # a vocabulary of 16
    for bad in (-1, 16, 1 << 20):
        with pytest.raises(ValueError, match="token ids"):
            eng.step(bad)
    assert eng.launched == 0
    eng.step(15)
    eng.step(0)
    assert eng.launched == 2
