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
