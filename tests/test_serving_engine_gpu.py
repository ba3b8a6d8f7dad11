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


def _large_past(kv_bits):
    """A layer behind 10 cached positions whose values are around 3e5 and whose keys are 1e6 in two channels that no query
    has (both beyond fp16).  Queries are the biases alone, 0.02, so that scores are of size one."""
    from dataclasses import replace

    spec = replace(Q.TINY, L=1)
    w = Q.build(spec)
    p, hd = "model.layers.0.self_attn", spec.H // spec.NH
    w[f"{p}.q_proj.weight"] = np.zeros_like(w[f"{p}.q_proj.weight"])
    rng = np.random.default_rng(8)
    bias = (0.02 * rng.standard_normal((spec.NH, hd))).astype(np.float32)
    bias[:, [31, 63]] = 0.0
    w[f"{p}.q_proj.bias"] = bias.reshape(-1)
    for m in ("k", "v"):
        w[f"{p}.{m}_proj.bias"] = np.zeros(spec.NKV * hd, np.float32)
    k, v = (rng.standard_normal((10, spec.NKV, hd)).astype(np.float32) for _ in range(2))
    k[:, :, 31], k[:, :, 63] = 1e6, -1e6
    v = (3e5 + 1e5 * v).astype(np.float32)
    return _engine(spec=spec, weights=w, kv_bits=kv_bits, kv_page=16, kv_prefill={0: (k, v)})


@pytest.mark.parametrize("bits", [32, 4])
def test_prefill_behind_values_beyond_fp16(bits):
    """A prompt at once gives what its tokens give one by one.  fp16 roundings between the two: of queries, keys, weights,
    values, the attention's result, and two operands of each batched product, 2^-11 each: below 16 * 2^-11 of the logits'
    size.  (In 4 bits the prompt's own keys differ too, exact in one and quantised in the other: finite is all that is asked.)"""
    tokens = np.random.default_rng(3).integers(0, 320, 20)
    one, eng = _large_past(bits), _large_past(bits)
    for t in tokens:
        one.step(int(t))
    eng.prefill(tokens)
    ref, got = one.logits_host(), eng.logits_host()
    assert np.isfinite(ref).all() and np.isfinite(got).all()
    if bits == 32:
        assert np.abs(got - ref).max() <= 2.0 ** -7 * np.abs(ref).max()


@pytest.mark.parametrize("bits", [32, 4])
def test_capture_keeps_the_last_token(bits):
    """prefill, then capture: logits and pick are the prompt's still, and the pick goes in next, as without a capture."""
    tokens = np.random.default_rng(4).integers(0, 320, 23)
    plain, eng = _engine(kv_bits=bits), _engine(kv_bits=bits)
    for e in (plain, eng):
        e.prefill(tokens)
    logits, pick = eng.logits_host().copy(), eng.argmax_host()
    eng.capture()
    assert np.array_equal(eng.logits_host(), logits) and eng.argmax_host() == pick
    assert int(eng.pos.item()) == 23
    for _ in range(3):
        for e in (plain, eng):
            e.step()
        assert np.array_equal(eng.logits_host(), plain.logits_host()) and eng.argmax_host() == plain.argmax_host()


def test_launches_of_a_token():
    """The count of a token's kernels stays through a prompt; a layer whose attention needs no join has one less (2 KV heads,
    each 3 places of 32 tokens and one: 8, which are a CTA's; with a fourth place 10)."""
    counts = []
    for max_pos in (96, 97):
        eng = _engine(max_pos=max_pos, kv_bits=4, kv_page=16)
        eng.capture()
        counts.append(eng.launches_per_token)
        eng.prefill(np.arange(20))
        assert eng.launches_per_token == counts[-1]
        eng.step()
        assert eng.launches_per_token == counts[-1]
    assert counts[1] - counts[0] == Q.TINY.L


def test_outputs_in_place_and_beside():
    """Decode attention into its queries and into columns of their buffer gives what it gives into memory of its own; an
    output that lies over them by a part is refused."""
    from flatrun_b200 import attention as A

    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    lens = [700, 3, 0, 5000]
    cache = A.kv_cache_q4(100, 64, 2, 128)
    k, v = (torch.randn((6400, 2, 128), generator=g, device="cuda") for _ in range(2))
    A.kv_append_q4(cache, k, v, torch.arange(6400, device="cuda"))
    table = torch.arange(100, dtype=torch.int32, device="cuda").repeat(4, 1)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for heads in (4, 32):
        buffer = torch.zeros((4, 2 * heads, 128), device="cuda")
        q, beside = buffer[:, :heads], buffer[:, heads:]
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        ref = A.attention_decode_q4(q, cache, table, n)
        for _ in range(5):
            again = q.clone()
            A.attention_decode_q4(q, cache, table, n, out=beside)
            A.attention_decode_q4(again, cache, table, n, out=again)
            assert torch.equal(beside, ref) and torch.equal(again, ref)
        with pytest.raises(ValueError, match="share"):
            A.attention_decode_q4(q, cache, table, n, out=buffer[:, 1:heads + 1])
        with pytest.raises(ValueError, match="finite"):
            A.attention_decode_q4(q, cache, table, n, scale=float("nan"))


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("parts", [(33,), (1, 5), (20, 17), (16, 40, 9)])
def test_prefill_attention_of_every_layer(bits, parts, monkeypatch):
    """What each layer's prompt attention is given and gives.  Keys and values are the cache's of the past and behind them
    the prompt's own, which are the ones that the cache takes; the result is that of the 64-bit restatement."""
    import test_attention_gpu as T
    from flatrun_b200 import attention as A

    calls = []
    real = A.attention_prefill

    def recorded(q, k, v, cu_q, cu_k, **kw):
        out = real(q, k, v, cu_q, cu_k, **kw)
        calls.append((q.clone(), k.clone(), v.clone(), cu_q.tolist(), cu_k.tolist(), out.clone()))
        return out

    monkeypatch.setattr(A, "attention_prefill", recorded)
    rng = np.random.default_rng(sum(parts))
    eng = _engine(kv_bits=bits, kv_page=16)

    def cached(layer, n):
        if bits == 32:
            return eng.k_cache[layer][:n].clone(), eng.v_cache[layer][:n].clone()
        return A.kv_read_q4(eng.q4_cache[layer], torch.arange(n, device="cuda"))

    start = 0
    for n in parts:
        eng.stream.synchronize()
        past = [cached(i, start) for i in range(Q.TINY.L)]
        calls.clear()
        eng.prefill(rng.integers(0, 320, n))
        eng.stream.synchronize()
        assert len(calls) == Q.TINY.L
        for i, (q, k, v, cu_q, cu_k, out) in enumerate(calls):
            assert cu_q == [0, n] and cu_k == [0, start + n]
            for x, before, after in zip((k, v), past[i], cached(i, start + n)):
                assert torch.equal(x[:start], before.half())
                if bits == 32:
                    assert torch.equal(x[start:], after[start:].half())
                else:  # fp16's rounding and the cache's: half a step, and the roundings of d and m
                    own = T._np(after[start:])
                    _, d, _ = T.R.quantise(T._np(x[start:]))
                    bound = np.repeat(d, 32, -1) * (0.5 + 16 * 2.0 ** -11) + np.abs(T._np(x[start:])).max() * 2.0 ** -10
                    T._close(x[start:], own, bound)
            ref, bound = T._prefill_ref(T._np(q), T._np(k), T._np(v), cu_q, cu_k, True, float(np.float32(0.125)), "fp16")
            T._close(out, ref, bound)
        start += n
    assert int(eng.pos.item()) == start
    if bits == 4:
        assert int(eng._slot.item()) == start and int(eng._length.item()) == start + 1
        # the next token lies behind the prompts and attends over all of them
        eng.step(7)
        eng.stream.synchronize()
        q = eng.qkv[:eng.cfg.hidden].view(1, -1, 64)
        o, bound = T._decode_ref(eng.q4_cache[-1], eng._table, torch.tensor([start + 1]), T._np(q), 0.125, "fp32", 16)
        T._close(eng.ctx.view(1, -1, 64), o, bound)


def test_prefill_behind_a_4_bit_past_equals_one_behind_the_same_in_fp32():
    """An fp32 engine that starts from what a 4-bit one holds gives the same logits for the next prompt, bit for bit."""
    from flatrun_b200 import attention as A

    rng = np.random.default_rng(9)
    first, second = rng.integers(0, 320, 21), rng.integers(0, 320, 18)
    four = _engine(kv_bits=4, kv_page=16)
    four.prefill(first)
    four.stream.synchronize()
    at = torch.arange(21, device="cuda")
    past = {i: tuple(x.cpu().numpy() for x in A.kv_read_q4(c, at)) for i, c in enumerate(four.q4_cache)}
    full = _engine(kv_prefill=past)
    for e in (four, full):
        e.prefill(second)
    assert np.array_equal(four.logits_host(), full.logits_host())
    assert four.argmax_host() == full.argmax_host()


@pytest.mark.parametrize("bits", [32, 4])
def test_construction_is_over_when_it_returns(bits):
    """Weights, zeroed buffers and a stored past are there before the engine's own stream can touch them."""
    kv = {i: (np.ones((40, Q.TINY.NKV, 64), np.float32),) * 2 for i in range(Q.TINY.L)}
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            _engine(kv_bits=bits, kv_prefill=kv)
            assert side.query()
