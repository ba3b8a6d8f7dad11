"""The decode engine's serving paths (GPU): the ends of the cache, prompts, captured tokens."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import qwen2_restated as Q

pytestmark = pytest.mark.gpu


def _engine(max_pos=100, spec=Q.TINY, weights=None, **kw):
    from flatrun_b200.decode import DecodeEngine, DecoderConfig

    s = spec
    cfg = DecoderConfig(s.H, s.F, s.V, s.L, s.NH, s.NKV, s.EPS, s.THETA, max_pos)
    return DecodeEngine(cfg, Q.build(s) if weights is None else weights, lambda name: Q.quant_of(s, name), **kw)


@pytest.mark.parametrize("bits", [32, 4])
def test_the_last_position_is_used_and_none_behind_it(bits):
    """21 positions (in 4 bits: in two pages of 16): a prompt of 20 and a token fill them; step, capture and prefill
    then raise, and what was computed stays."""
    eng = _engine(max_pos=21, kv_bits=bits, kv_page=16)
    eng.prefill(np.arange(20))
    eng.step(5)
    logits = eng.logits_host().copy()
    assert np.isfinite(logits).all() and int(eng.pos.item()) == 21
    for call in (lambda: eng.step(1), eng.step, eng.capture, lambda: eng.prefill([1])):
        with pytest.raises(ValueError, match="max_pos"):
            call()
    assert np.array_equal(eng.logits_host(), logits) and int(eng.pos.item()) == 21
    kv = {0: (np.zeros((22, Q.TINY.NKV, 64), np.float32),) * 2}
    with pytest.raises(ValueError, match="max_pos"):
        _engine(max_pos=21, kv_bits=bits, kv_page=16, kv_prefill=kv)
