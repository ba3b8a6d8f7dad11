"""The serving operators restated in NumPy and 64 bits, one statement at a
time from their definitions: the oracle of their tests.  Nothing here shares
code with the package."""

from __future__ import annotations

import numpy as np

HALF = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def half_grid(x):
    """x >= 0 (fp64) at the nearest fp16 value, ties to even, at most 65504."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(x)
    ulp = np.ldexp(1.0, np.maximum(e - 11, -24))
    return np.minimum(np.rint(x / ulp) * ulp, 65504.0)


def quantise(x):
    """x (..., D) -> n (..., D) uint8, d and m (..., D / 32) as fp64 values of fp16."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        ok = np.isfinite(g).all(-1)
        low, high = g.min(-1), g.max(-1)
        m = np.clip(low, -65504.0, 65504.0).astype(np.float32).astype(np.float16).astype(np.float64)
        d = half_grid(np.where(ok, np.maximum(high - m, 0.0) / 15.0, 0.0))
        n = np.where(d[..., None] > 0, np.clip(np.rint((g - m[..., None]) / np.where(d > 0, d, 1.0)[..., None]), 0, 15), 0)
    n = np.where(ok[..., None], n, 0).astype(np.uint8)
    return n.reshape(x.shape), d, np.where(ok, m, np.nan)


def value(n, d, m):
    """d * n + m, in 64 bits."""
    return (n.reshape(*n.shape[:-1], -1, 32) * d[..., None] + m[..., None]).reshape(n.shape)


def _places(hd):
    """Byte and shift of every nibble, and byte of every scale, in a block of 16 tokens."""
    ng = hd // 32
    t, c = np.meshgrid(np.arange(16), np.arange(hd), indexing="ij")
    j, q, i = c // 32, c % 32 // 8, c % 8
    k = 4 * ((t * 4 + q) * ng + j) + i // 2
    v = 8 * hd + 4 * ((c // 8) * 16 + t) + i // 2
    t, j = np.meshgrid(np.arange(16), np.arange(ng), indexing="ij")
    scales = (16 * hd + 2 * (16 * j + t), 17 * hd + 2 * (ng * t + j), 18 * hd + 2 * (16 * j + t),
              19 * hd + 2 * (16 * j + t))
    return k, v, i % 2, scales


def unpack(cache):
    """A cache (pages, heads, blocks, 20 hd) -> K and V (pages, heads, page_size, hd) values in
    64 bits, and the sums |d n| + |m| of each."""
    pages, heads, blocks, nbytes = cache.shape
    hd = nbytes // 20
    kb, vb, odd, scales = _places(hd)
    flat = cache.reshape(-1, nbytes)
    kd, km, vd, vm = ((flat[:, s].astype(np.uint16) | (flat[:, s + 1].astype(np.uint16) << 8)).view(np.float16)
                      .astype(np.float64) for s in scales)
    out = []
    for b, d, m in ((kb, kd, km), (vb, vd, vm)):
        n = ((flat[:, b] >> (4 * odd)) & 15).astype(np.float64)
        d, m = np.repeat(d, 32, axis=-1), np.repeat(m, 32, axis=-1)
        for x in (n * d + m, n * np.abs(d) + np.abs(m)):
            out.append(x.reshape(pages, heads, blocks * 16, hd))
    return out[0], out[2], out[1], out[3]


def middle_sizes(cache):
    """|d (n - 8)| + |m + 8 d| of V (pages, heads, page_size, hd): the terms of a value taken from its group's middle."""
    pages, heads, blocks, nbytes = cache.shape
    hd = nbytes // 20
    _, at, odd, scales = _places(hd)
    flat = cache.reshape(-1, nbytes)
    d, m = ((flat[:, s].astype(np.uint16) | (flat[:, s + 1].astype(np.uint16) << 8)).view(np.float16)
            .astype(np.float64).repeat(32, axis=-1) for s in scales[2:])
    n = ((flat[:, at] >> (4 * odd)) & 15).astype(np.float64)
    return (np.abs(d * (n - 8)) + np.abs(m + 8 * d)).reshape(pages, heads, blocks * 16, hd)


def write(cache, k, v, slots):
    """Quantise rows into a cache (uint8, changed in place); slots outside it are skipped."""
    pages, heads, blocks, nbytes = cache.shape
    kb, vb, odd, scales = _places(nbytes // 20)
    for i, slot in enumerate(slots):
        if not 0 <= slot < pages * blocks * 16:
            continue
        page, at = divmod(int(slot), blocks * 16)
        for h in range(heads):
            blk, t = cache[page, h, at // 16], at % 16
            for x, b, sd, sm in ((k[i, h], kb, scales[0], scales[1]), (v[i, h], vb, scales[2], scales[3])):
                n, d, m = quantise(x)
                blk[b[t]] = 0  # both nibbles of a byte belong to the token
                np.bitwise_or.at(blk, b[t], (n << (4 * odd[t])).astype(np.uint8))
                for place, s in ((sd, d), (sm, m)):
                    raw = s.astype(np.float16)
                    raw[np.isnan(s)] = np.array(0x7FFF, np.uint16).view(np.float16)
                    raw = raw.view(np.uint16)
                    blk[place[t]], blk[place[t] + 1] = raw & 255, raw >> 8


def rope(x, heads, kv_heads, cos, sin, pos, bias=None, q_norm=None, k_norm=None, eps=1e-6, interleaved=False):
    """rows (T, n) -> q, k, v in 64 bits, and for each the size |a| + |b| that roundings of it scale with."""
    t, n = x.shape
    hd = n // (heads + 2 * kv_heads)
    x = x.astype(np.float64) + (0 if bias is None else bias.astype(np.float64))
    x = x.reshape(t, -1, hd)
    rot = 2 * cos.shape[1]
    first = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    c, s = cos.astype(np.float64)[pos][:, None], sin.astype(np.float64)[pos][:, None]
    out = []
    for h, w in ((x[:, :heads], q_norm), (x[:, heads:heads + kv_heads], k_norm)):
        if w is not None:
            h = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        y, size = h.copy(), np.abs(h)
        a, b = h[..., first], h[..., second]
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        size[..., first] = size[..., second] = (np.abs(a) + np.abs(b)) * np.maximum(np.abs(c), np.abs(s))
        out.append((y, size))
    v = x[:, heads + kv_heads:]
    return [*out, (v, np.abs(v))]


def attend(q, k, v, scale, seen=None):
    """softmax(scale q k^T) v over the seen keys (zeros where there is none), and sum p |v|: q (H, D) or
    (N, D), k and v (T, D), all 64 bits."""
    s = q @ k.T * scale
    if seen is not None:
        s = np.where(seen, s, -np.inf)
    if s.size == 0:
        return np.zeros_like(q), np.zeros_like(q)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdims=True)
    p = p / np.where(total > 0, total, 1.0)
    if seen is not None:  # what is masked has no part in the result, whatever it holds
        rows = [np.where(seen[i], p[i], 0.0)[seen[i]] @ v[seen[i]] for i in range(len(p))]
        return np.stack(rows), np.stack([p[i][seen[i]] @ np.abs(v[seen[i]]) for i in range(len(p))])
    return p @ v, p @ np.abs(v)
