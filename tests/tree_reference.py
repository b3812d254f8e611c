"""Plain 64-bit forms of the operators of a step that verifies drafted tokens -- norms with rotary positions,
e4m3 cache rows, attention under token masks -- and the bounds their kernels keep (see
packed_reference.py for how a bound adds up)."""
from __future__ import annotations

import numpy as np

from tests.packed_reference import FP32, HALF_STEP, rope

LOWEST, HIGHEST = -64, 32  # exponents of an e4m3 head row

# the 127 values from 0 up to 448, by their codes
_MAGNITUDES = np.array([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10)
                        for c in range(127)])


def e4m3_codes(x):
    """float64 values -> codes, to nearest, ties to the even code; beyond 448: 448; not finite: NaN."""
    a = np.minimum(np.abs(np.where(np.isfinite(x), x, 0.0)), 448.0)
    up = np.searchsorted(_MAGNITUDES, a).clip(1, 126)
    lo, hi = a - _MAGNITUDES[up - 1], _MAGNITUDES[up] - a
    code = np.where((lo < hi) | ((lo == hi) & ((up - 1) % 2 == 0)), up - 1, up)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(np.isfinite(x), code, 0x7F).astype(np.uint8)


def e4m3_values(codes):
    m = np.concatenate([_MAGNITUDES, [np.nan]])[codes & 0x7F]
    return np.where(codes & 0x80, -m, m)


def quantise(x):
    """Head rows [..., d] in 64 bits -> (codes [..., d], exponents [...])."""
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    m, k = np.frexp(top)  # m in [0.5, 1): 448 = 0.875 * 2^9
    e = np.where(top == 0, LOWEST, k - 9 + (m > 0.875)).clip(LOWEST, HIGHEST)
    return e4m3_codes(np.ldexp(x, -e[..., None])), e.astype(np.int64)


def dequantise(codes, e):
    return np.ldexp(e4m3_values(codes), e[..., None])


def norm_rope(x, gain, eps, positions, axis, freq, rotary, interleaved, amplitude, dtype):
    """x [T][heads][d] in 64 bits, gain [d] or None, positions [axes][T], axis [rotary / 2] -> (y, bound)."""
    u = HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    d = x.shape[2]
    z, loose = x, 0.0
    if gain is not None:
        z = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * gain
        # half the error of a sum of d squares, a root, two quotients, three products
        loose = ((d + 2) / 2 + 8) * FP32
    if rotary == 0:
        return z, np.abs(z) * (loose + u * (1 + loose)) + tiny
    y, bound = z.copy(), np.abs(z) * (loose + u * (1 + loose)) + tiny
    for a in np.unique(axis):
        # (one axis after the other: the pairs of the others are left out of what it gives)
        at = positions[a] if a < len(positions) else np.zeros_like(positions[0])
        ya, ba = rope(z, at, freq, rotary, interleaved, amplitude, "f32")
        pairs = np.nonzero(axis == a)[0]
        i = 2 * pairs if interleaved else pairs
        j = i + 1 if interleaved else i + rotary // 2
        size = (np.abs(z[..., i]) + np.abs(z[..., j])) * amplitude * loose
        for e in (i, j):
            y[..., e] = ya[..., e]
            off = ba[..., e] + size
            bound[..., e] = off + u * (np.abs(ya[..., e]) + off) + tiny
    return y, bound


def ancestors(parents):
    """bool [n][n]: the row's own token and its ancestors."""
    n = len(parents)
    seen = np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] |= seen[p]
    return seen


def mask_bits(seen, words):
    bits = np.zeros((seen.shape[0], 64 * words), np.uint8)
    bits[:, :seen.shape[1]] = seen
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint64)


def tree_attention(q, k, v, seen, scale, dtype, k_exp=None, v_exp=None):
    """One sequence: q [n][hq][d], k and v [ctx][hkv][d] in 64 bits, seen bool [n][ctx]; exponents [ctx][hkv] of
    e4m3 rows -> (out, bound).  What is not seen does not enter."""
    n, hq, d = q.shape
    ctx, hkv = k.shape[:2]
    g, u = hq // hkv, HALF_STEP[dtype]
    out, bound = np.zeros(q.shape), np.full(q.shape, 2.0 ** -25 if dtype == "fp16" else 0.0)
    if ctx == 0:
        return out, bound

    def step(e):  # half a step of fp16 below its range, relative to the largest exponent of 32 neighbours
        top = np.repeat([e[i:i + 32].max(0) for i in range(0, ctx, 32)], 32, 0)[:ctx]
        return 2.0 ** (top - 25.0)

    for h in range(hq):
        kh, vh = k[:, h // g], v[:, h // g]
        clean_k, clean_v = np.where(seen.any(0)[:, None], kh, 0.0), np.where(seen.any(0)[:, None], vh, 0.0)
        s = (q[:, h] @ clean_k.T) * scale
        size = (np.abs(q[:, h]) @ np.abs(clean_k).T) * scale
        off = (d + 6) * FP32 * size
        if k_exp is not None and dtype == "fp16":
            off = off + np.abs(q[:, h]).sum(1, keepdims=True) * step(k_exp)[:, h // g] * scale
        s, off = np.where(seen, s, -np.inf), np.where(seen, off, 0.0)
        top = s.max(1, keepdims=True)
        some = np.isfinite(top[:, 0])
        w = np.exp(s - np.where(some[:, None], top, 0.0))
        p = w / np.where(some, w.sum(1), 1.0)[:, None]
        o, mean = p @ clean_v, p @ np.abs(clean_v)
        reach = np.where(np.isinf(s), 0, np.where(some[:, None], top, 0.0) - s).max(1, keepdims=True)
        delta = off.max(1, keepdims=True) + 4 * FP32 * (reach + 16) + 4 * 2.0 ** -22
        # (a probability enters the product to half a step of fp16, or to 2^-36 of the largest, which is at least 1 / w.sum())
        lost = ctx * 2.0 ** -36 * np.abs(clean_v).max(0)[None]
        if v_exp is not None:
            lost = lost + (p @ step(v_exp)[:, h // g])[:, None] + \
                ctx * 2.0 ** -36 * 448 * 2.0 ** np.where(seen.any(0), v_exp[:, h // g], -99).max()
        e = 2.0 ** -11 * mean + 2 * delta * mean + 2 * ctx * FP32 * mean + lost
        out[:, h] = np.where(some[:, None], o, 0.0)
        bound[:, h] += np.where(some[:, None], u * np.abs(o) * (1 + u) + e * (1 + 4 * u), 0.0)
    return out, bound
