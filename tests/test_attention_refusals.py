"""What the serving operators refuse, before anything is launched, and the
parts of them that need no GPU (rotation tables, cache sizes)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from flatrun_b200 import _lib, attention as A
import q4_restated as R


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from flatrun_b200 import build
        build.build()
    return _lib.load()


def _rope_args(**over):
    a = dict(qkv=torch.zeros(3, 8 * 64), heads=4, kv_heads=2, cos=torch.zeros(9, 32), sin=torch.zeros(9, 32),
             positions=torch.zeros(3, dtype=torch.int32))
    a.update(over)
    return a


@pytest.mark.parametrize("over,msg", [
    (dict(qkv=torch.zeros(3, 8 * 64, dtype=torch.float64)), "qkv"),
    (dict(qkv=torch.zeros(8 * 64)), "2-D"),
    (dict(heads=5), "do not hold"),
    (dict(heads=0), "positive"),
    (dict(qkv=torch.zeros(3, 8 * 63)), "even"),
    (dict(qkv=torch.zeros(3, 8 * 258)), "at most 256"),
    (dict(qkv=torch.zeros(8 * 64, 3).T), "contiguous"),
    (dict(cos=torch.zeros(9, 33), sin=torch.zeros(9, 33)), "rotate 66"),
    (dict(sin=torch.zeros(9, 31)), "one shape"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions"),
    (dict(bias=torch.zeros(7)), "bias"),
    (dict(q_norm=torch.zeros(64, dtype=torch.float16)), "q_norm"),
    (dict(out_dtype=torch.float64), "out_dtype"),
    (dict(out=(torch.zeros(3, 4, 64), torch.zeros(3, 2, 64))), "out"),
    (dict(out=(torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(2, 2, 64))), "out v"),
    (dict(out=(torch.zeros(3, 64, 4).transpose(1, 2), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64))), "channels"),
    (dict(), "CUDA device"),
])
def test_rope_refusals(over, msg):
    with pytest.raises(ValueError, match=msg):
        A.qk_norm_rope(**_rope_args(**over))


def test_gradients_are_refused():
    with pytest.raises(ValueError, match="no backward"):
        A.qk_norm_rope(**_rope_args(qkv=torch.zeros(3, 8 * 64, requires_grad=True)))


def test_cache_refusals():
    for kw, msg in ((dict(pages=0), "positive"), (dict(page_size=24), "multiple of 16"), (dict(head_dim=96), "64 or 128")):
        with pytest.raises(ValueError, match=msg):
            A.kv_cache_q4(**{**dict(pages=2, page_size=16, kv_heads=2, head_dim=64, device="cpu"), **kw})
    cache = A.kv_cache_q4(2, 32, 2, 64, device="cpu")
    assert cache.shape == (2, 2, 2, 1280)
    k, slots = torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int64)
    for a, msg in (((cache[..., :-1], k, k, slots), "cache"), ((cache, k[:, :1], k, slots), "k must"),
                   ((cache, k, k[:4], slots), "v must"), ((cache, k, k.half(), slots), "v must"),
                   ((cache, k, k, slots.int()), "slots"), ((cache, k.double(), k.double(), slots), "keys"),
                   ((cache, torch.zeros(5, 64, 2).transpose(1, 2), k, slots), "channels"),
                   ((cache, k, k, slots), "CUDA device")):
        with pytest.raises(ValueError, match=msg):
            A.kv_append_q4(*a)
    for kw, msg in ((dict(dtype=torch.float64), "dtype"), (dict(out=(k, k[:4])), "out v"), (dict(out=(k,)), "out"),
                    (dict(out=(k, k), dtype=torch.float16), "type asked"), (dict(), "CUDA device")):
        with pytest.raises(ValueError, match=msg):
            A.kv_read_q4(cache, slots, **kw)


def test_decode_refusals():
    cache = A.kv_cache_q4(2, 32, 2, 64, device="cpu")
    q, table, n = torch.zeros(3, 4, 64), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for a, msg in (((q[:, :3], cache, table, n), "multiple of"), ((q[..., :32], cache, table, n), "q must"),
                   ((q.double(), cache, table, n), "q must"), ((q, cache, table[:2], n), "block_table"),
                   ((q, cache, table.long(), n), "block_table"), ((q, cache, table, n.long()), "lengths"),
                   ((q, cache.view(-1), table, n), "cache"), ((q, cache, table, n), "CUDA device")):
        with pytest.raises(ValueError, match=msg):
            A.attention_decode_q4(*a)
    with pytest.raises(ValueError, match="out"):
        A.attention_decode_q4(q, cache, table, n, out=q.half())


def test_prefill_refusals():
    q, k = torch.zeros(5, 4, 64, dtype=torch.float16), torch.zeros(5, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 5], dtype=torch.int32)
    for a, msg in (((q.float(), k, k, cu), "fp16 or bf16"), ((q, k.bfloat16(), k, cu), "k must"),
                   ((q, k, k[:4], cu), "v must"), ((q[:, :3], k, k, cu), "multiple of"),
                   ((q[..., :32], k[..., :32], k[..., :32], cu), "64 or 128"), ((q, k, k, cu.long()), "cu_q"),
                   ((q, k, k, cu, cu[:1]), "cu_k"), ((q, k, k, cu[:0]), "ends"),
                   ((torch.zeros(5 * 4 * 64 + 1, dtype=torch.float16)[1:].view(5, 4, 64), k, k, cu), "aligned"),
                   ((torch.zeros(5, 4, 68, dtype=torch.float16)[..., :64], k, k, cu), "multiples of 8"),
                   ((q, k, k, cu), "CUDA device")):
        with pytest.raises(ValueError, match=msg):
            A.attention_prefill(*a)
    with pytest.raises(ValueError, match="out must not be"):
        A.attention_prefill(q, k, k, cu, out=q)


def test_c_abi_refusals(lib):
    """The C entry points check before any CUDA call."""
    p16 = ctypes.c_void_p(16)
    nb = ctypes.c_size_t()
    assert lib.frc_kv_q4_bytes(3, 32, 2, 64, ctypes.byref(nb)) == 0 and nb.value == 3 * 2 * 2 * 1280
    for bad in ((0, 32, 2, 64), (3, 24, 2, 64), (3, 32, 0, 64), (3, 32, 2, 96), (1 << 31, 16, 1, 64)):
        assert lib.frc_kv_q4_bytes(*bad, ctypes.byref(nb)) == _lib.FRC_ERR_INVALID

    def append(type=0, k=p16, k_tok=128, tokens=4, nkv=2, hd=64, pages=3, page=32, cache=p16):
        return lib.frc_kv_append_q4(type, k, k_tok, 64, p16, 128, 64, tokens, p16, nkv, hd, pages, page, cache, None)

    for kw in (dict(type=8), dict(k=None), dict(k_tok=-1), dict(tokens=-1), dict(nkv=0), dict(hd=96), dict(pages=0),
               dict(page=8), dict(cache=ctypes.c_void_p(8)), dict(pages=1 << 40)):
        assert append(**kw) == _lib.FRC_ERR_INVALID, kw
        assert "kv_q4" in _lib.last_error(lib)
    assert append(tokens=0, k=None) == 0

    def rope(hd=64, rot=64, stride=512, types=(0, 0), qkv=p16, max_pos=10):
        return lib.frc_qk_norm_rope(*types, qkv, stride, 2, 4, 2, hd, None, None, None, 1e-6, p16, p16, max_pos, rot, 0,
                                    p16, p16, 256, p16, 128, p16, 128, None)

    for kw in (dict(hd=63), dict(hd=258), dict(rot=66), dict(rot=3), dict(stride=511), dict(types=(0, 8)),
               dict(qkv=None), dict(max_pos=0)):
        assert rope(**kw) == _lib.FRC_ERR_INVALID, kw

    def decode(hd=64, nh=4, page=32, ws=1 << 30, q=p16, cache=p16, batch=2, table=p16, scale=0.1):
        return lib.frc_attention_decode_q4(0, q, 256, 64, cache, 3, page, table, 2, 2, p16, batch, nh, 2, hd, scale, p16,
                                           ws, p16, 256, 64, None)

    for kw in (dict(hd=96), dict(nh=5), dict(page=20), dict(ws=0), dict(q=None), dict(cache=ctypes.c_void_p(24)),
               dict(batch=-1), dict(table=None), dict(scale=math.inf), dict(scale=math.nan)):
        assert decode(**kw) == _lib.FRC_ERR_INVALID, kw
    assert decode(batch=0, q=None) == 0

    def prefill(type=1, hd=64, nh=4, stride=256, q=p16):
        return lib.frc_attention_prefill(type, q, stride, 64, p16, 128, 64, p16, 128, 64, p16, p16, 1, 5, 5, nh, 2, hd, 0.1,
                                         1, p16, 256, 64, None)

    for kw in (dict(type=0), dict(hd=96), dict(nh=5), dict(stride=252), dict(stride=-8), dict(q=None),
               dict(q=ctypes.c_void_p(8))):
        assert prefill(**kw) == _lib.FRC_ERR_INVALID, kw


def test_rope_tables():
    """Unscaled: the angle of every position in 64 bits.  Each scaling against its formula at single pairs."""
    cos, sin = A.rope_tables_scaled(64, 1e4, 200000)
    for i, p in ((0, 199999), (5, 131071), (31, 7)):
        a = p * 1e4 ** (-2 * i / 64)
        assert abs(cos[p, i] - math.cos(a)) <= 1e-7 and abs(sin[p, i] - math.sin(a)) <= 1e-7

    def angles(scaling):  # inverse frequencies from position 1, angles at most 1
        c, s = A.rope_tables_scaled(64, 1e4, 2, scaling)
        return np.arctan2(s[1], c[1]), np.hypot(c[1], s[1])

    inv = 1e4 ** (-np.arange(32) / 32)
    got, mag = angles({"type": "linear", "factor": 4})
    np.testing.assert_allclose(got, inv / 4, rtol=3e-7)
    np.testing.assert_allclose(mag, 1, rtol=3e-7)
    got, _ = angles({"type": "ntk", "factor": 4})
    np.testing.assert_allclose(got[[0, 31]], [1, inv[31] / 4], rtol=3e-7)
    got, mag = angles({"type": "yarn", "factor": 4, "original_max_position": 4096})
    np.testing.assert_allclose(got[[0, 31]], [1, inv[31] / 4], rtol=3e-7)
    np.testing.assert_allclose(mag, 0.1 * math.log(4) + 1, rtol=3e-7)
    assert np.all(np.diff(got) < 0)
    got, mag = angles({"type": "llama3", "factor": 8, "original_max_position": 8192})
    turns = 8192 * inv / (2 * math.pi)
    np.testing.assert_allclose(got[turns > 4], inv[turns > 4], rtol=3e-7)
    np.testing.assert_allclose(got[turns < 1], inv[turns < 1] / 8, rtol=3e-7)
    mid = (turns > 1) & (turns < 4)
    keep = (turns[mid] - 1) / 3
    np.testing.assert_allclose(got[mid], (1 - keep) * inv[mid] / 8 + keep * inv[mid], rtol=3e-7)
    for bad in ({"type": "spiral", "factor": 2}, {"type": "linear", "factor": 0.5}, {"type": "yarn", "factor": 2},
                {"type": "llama3", "factor": 2, "original_max_position": 0}):
        with pytest.raises(ValueError):
            A.rope_tables_scaled(64, 1e4, 4, bad)
    with pytest.raises(ValueError, match="theta"):
        A.rope_tables_scaled(64, 1.0, 4, {"type": "yarn", "factor": 2, "original_max_position": 64})


def test_oracle_of_the_cache_round_trips():
    """The restated cache: what is written reads back as d * n + m within half a step, and NaN for groups that are not finite."""
    rng = np.random.default_rng(0)
    for hd in (64, 128):
        cache = np.zeros((2, 2, 2, 20 * hd), np.uint8)
        k, v = (rng.standard_normal((5, 2, hd)).astype(np.float32) for _ in range(2))
        k[2, 1, 40] = np.inf
        slots = np.array([3, 63, -1, 17, 64])
        slots[2] = 40
        R.write(cache, k, v, slots)
        kk, vv, _, _ = R.unpack(cache)
        kk, vv = (x.transpose(0, 2, 1, 3).reshape(64, 2, hd) for x in (kk, vv))
        for i in (0, 1, 3):
            for x, y in ((k[i], kk[slots[i]]), (v[i], vv[slots[i]])):
                _, d, _ = R.quantise(x)
                # half a step, and the roundings of d and m to fp16: 15 n d off by 2^-11, m by 2^-11
                bound = np.repeat(d, 32, -1) * (0.5 + 15 * 2.0 ** -11) + np.abs(x).max() * 2.0 ** -11
                assert np.all(np.abs(x - y) <= bound)
        assert np.isnan(kk[40, 1, 32:64]).all() and np.isfinite(kk[40, 1, :32]).all() and np.isfinite(vv[40]).all()


def _calls():
    """Each operator with CPU tensors: (name of each floating tensor, the call with some of them replaced)."""
    half = torch.float16
    cache = A.kv_cache_q4(2, 32, 2, 64, device="cpu")
    slots, n = torch.zeros(5, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    rows = {"k": torch.zeros(5, 2, 64), "v": torch.zeros(5, 2, 64)}
    rope = {"qkv": torch.zeros(3, 512), "cos": torch.zeros(9, 32), "sin": torch.zeros(9, 32), "bias": torch.zeros(512),
            "q": torch.zeros(3, 4, 64), "k": torch.zeros(3, 2, 64), "v": torch.zeros(3, 2, 64)}
    decode = {"q": torch.zeros(3, 4, 64), "out": torch.zeros(3, 4, 64)}
    prefill = {"q": torch.zeros(5, 4, 64, dtype=half), "k": torch.zeros(5, 2, 64, dtype=half),
               "v": torch.zeros(5, 2, 64, dtype=half), "out": torch.zeros(5, 4, 64, dtype=half)}
    cu = torch.tensor([0, 5], dtype=torch.int32)
    return [
        (rope, lambda a: A.qk_norm_rope(a["qkv"], 4, 2, a["cos"], a["sin"], n, bias=a["bias"], out=(a["q"], a["k"], a["v"]))),
        (rows, lambda a: A.kv_append_q4(cache, a["k"], a["v"], slots)),
        (rows, lambda a: A.kv_read_q4(cache, slots, out=(a["k"], a["v"]))),
        (decode, lambda a: A.attention_decode_q4(a["q"], cache, n[:, None], n, out=a["out"])),
        (prefill, lambda a: A.attention_prefill(a["q"], a["k"], a["v"], cu, out=a["out"])),
    ]


@pytest.mark.parametrize("operator", range(5))
def test_derivatives_of_either_mode_are_refused(operator):
    """Inputs and outputs that require gradients, and inputs and outputs with tangents; without either the call gets as
    far as the device."""
    from torch.autograd import forward_ad

    tensors, call = _calls()[operator]
    with pytest.raises(ValueError, match="CUDA device"):
        call(tensors)
    for name, t in tensors.items():
        with pytest.raises(ValueError, match="no backward"):
            call({**tensors, name: t.clone().requires_grad_()})
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call({**tensors, name: t.clone().requires_grad_()})
        with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            call({**tensors, name: forward_ad.make_dual(t, torch.ones_like(t))})
    with forward_ad.dual_level(), pytest.raises(ValueError, match="CUDA device"):
        call(tensors)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of no memory: where a GPU is, the calls below must not be launched")
def test_outputs_that_share_memory(lib):
    """The C entry points refuse outputs over inputs, over each other or over themselves.  What they take gets as far as the
    launch, which fails here without a device."""
    taken, refused = (_lib.FRC_ERR_CUDA,), (_lib.FRC_ERR_INVALID,)
    a = 1 << 20

    def prefill(out, o=(256, 64), q=a, q_strides=(256, 64), k=1 << 24, k_strides=(128, 64), tokens=5, nh=4):
        return lib.frc_attention_prefill(1, q, *q_strides, k, *k_strides, k + 8192, *k_strides, 16, 16, 1, tokens, 5, nh, 2, 64,
                                         0.1, 1, out, *o, None)

    far = 1 << 26
    row = dict(q_strides=(768, 64), k=a + 512, k_strides=(768, 64))  # [q 4 | k 2 | ...| out 4] heads of 64, 2 bytes each
    for rc, want in (
            (prefill(far), taken), (prefill(a + 16), refused), (prefill(a - 16), refused), (prefill(a + 5 * 512), taken),
            (prefill(a - 5 * 512), taken), (prefill(a), refused), (prefill((1 << 24) + 1024), refused),
            (prefill(a + 512, o=(768, 64), q_strides=(768, 64)), taken),      # columns of one buffer
            (prefill(a + 496, o=(768, 64), q_strides=(768, 64)), refused),
            (prefill(a + 5 * 128, o=(64, 640), q_strides=(64, 640)), taken),  # heads before tokens, by turns
            (prefill(a + 4 * 128, o=(64, 640), q_strides=(64, 640)), refused),
            (prefill(a + 128, o=(512, 128), q_strides=(512, 128)), taken),    # heads by turns
            (prefill(a + 112, o=(512, 128), q_strides=(512, 128)), refused),
            (prefill(far, o=(128, 64)), refused), (prefill(far, o=(0, 64)), refused), (prefill(far, o=(64, 320)), taken),
            (prefill(far, o=(64, 312)), refused), (prefill(far, o=(8, 64), tokens=1), taken),
            (prefill(far, o=(64, 8), q_strides=(64, 8), nh=2), refused),
            (prefill(far, **row), taken)):
        assert rc in want

    def decode(out, o=(256, 64), q=a, batch=3, cache=1 << 24):
        return lib.frc_attention_decode_q4(0, q, 256, 64, cache, 3, 32, 16, 2, 2, 16, batch, 4, 2, 64, 0.1, 1 << 28, 1 << 30, out,
                                           *o, None)

    for rc, want in ((decode(far), taken), (decode(a), taken), (decode(a + 16), refused), (decode(a, o=(512, 64)), refused),
                     (decode(a, o=(8, 64), batch=1), taken), (decode(a + 3 * 1024), taken), (decode(far, o=(192, 64)), refused),
                     (decode((1 << 24) + 3 * 2 * 2 * 1280), taken), (decode((1 << 24) + 3 * 2 * 2 * 1280 - 16), refused)):
        assert rc in want

    def read(k, v, strides=(128, 64), v_strides=None):
        return lib.frc_kv_read_q4(0, 1 << 24, 16, 5, 2, 64, 3, 32, k, *strides, v, *(v_strides or strides), None)

    for rc, want in ((read(a, far), taken), (read(a, a), refused), (read(a, a + 2560), taken), (read(a, a + 2556), refused),
                     (read(a, a + 256, (384, 192)), taken), (read(a, a + 128, (384, 192)), refused),
                     (read(a, far, (64, 64)), refused), (read(a, far, v_strides=(0, 64)), refused),
                     (read((1 << 24) + 1280, far), refused)):
        assert rc in want

    def rope(qkv, q, k, v, types=(0, 0), strides=(512, 512, 512, 512), tokens=3):
        return lib.frc_qk_norm_rope(*types, qkv, strides[0], tokens, 4, 2, 64, None, None, None, 1e-6, 16, 16, 10, 64, 0, 16, q,
                                    strides[1], k, strides[2], v, strides[3], None)

    own = (a, a, a + 1024, a + 1536)
    for rc, want in ((rope(*own), taken), (rope(*own, types=(0, 1)), refused), (rope(*own, strides=(512, 512, 520, 512)), refused),
                     (rope(*own, strides=(512, 256, 128, 128), tokens=1), taken), (rope(a, a, a + 1536, a + 1024), refused),
                     (rope(a, far, far + 1024, far + 1536), taken), (rope(a, far, far + 1024, far + 1024), refused),
                     (rope(a, far, far + 1020, far + 1536), refused), (rope(a, a, far, far + 512), refused),
                     (rope(a + 2048, a, far, far + 512, strides=(1024,) * 4), taken),
                     (rope(a + 1020, a, far, far + 512, strides=(1024,) * 4), refused)):
        assert rc in want


def test_operators_raise_value_errors(monkeypatch):
    """What the library refuses raises ValueError from the Python entry points, as what they refuse themselves does."""
    monkeypatch.setattr(A, "_device", lambda first, *others: 0)
    monkeypatch.setattr(A, "_current_device", lambda: 0)
    monkeypatch.setattr(A, "_raw_stream", lambda i: 0)
    q, k = torch.zeros(5, 4, 64, dtype=torch.float16), torch.zeros(5, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="scale must be finite"):
        A.attention_prefill(q, k, k, torch.tensor([0, 5], dtype=torch.int32), scale=math.inf)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of no memory: where a GPU is, the calls below must not be launched")
def test_numbers_of_sequences(lib):
    def prefill(batch):
        return lib.frc_attention_prefill(1, 1 << 20, 256, 64, 1 << 24, 128, 64, 1 << 25, 128, 64, 16, 16, batch, 5, 5, 4, 2, 64, 0.1,
                                         1, 1 << 26, 256, 64, None)

    assert prefill(1 << 20) == _lib.FRC_ERR_CUDA and prefill((1 << 20) + 1) == _lib.FRC_ERR_INVALID
