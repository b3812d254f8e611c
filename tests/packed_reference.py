"""Plain 64-bit forms of the operators over packed rows, and the bounds their kernels keep.

A bound adds up, element by element, what the documented arithmetic may lose: the rounding of the
result (half a step of its type, relative to it), the roundings of what goes into a product, and the
fp32 sums (a sum of n terms is off by at most n * 2^-24 times the sum of their magnitudes).
"""
from __future__ import annotations

import numpy as np

HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
FP32 = 2.0 ** -24


def to_bits(a, dtype):
    """float values -> what lies in memory (fp16, bf16 rounded to nearest even as uint16, f32)."""
    a = np.asarray(a, np.float32)
    if dtype == "f32":
        return a
    if dtype == "fp16":
        return a.astype(np.float16)
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), ((u >> 16) | 0x40).astype(np.uint16), r)


def from_bits(a, dtype):
    """... and back, in 64 bits."""
    if dtype == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def storage(dtype):
    return {"fp16": np.float16, "bf16": np.uint16, "f32": np.float32}[dtype]


def attention(q, k, v, lens, scale, causal, dtype):
    """q [T][hq][d], k and v [T][hkv][d] in 64 bits -> (out, bound)."""
    T, hq, d = q.shape
    g = hq // k.shape[1]
    u = HALF_STEP[dtype]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    at = 0
    for n in lens:
        r = slice(at, at + n)
        if n == 0:
            continue
        for h in range(hq):
            kh, vh = k[r, h // g], v[r, h // g]
            s = (q[r, h] @ kh.T) * scale
            size = (np.abs(q[r, h]) @ np.abs(kh).T) * scale
            if causal:
                hidden = np.triu(np.ones((n, n), bool), 1)
                s[hidden], size[hidden] = -np.inf, 0.0
            top = s.max(1, keepdims=True)
            w = np.exp(s - top)
            total = w.sum(1, keepdims=True)
            p = w / total
            o, mean = p @ vh, p @ np.abs(vh)
            # A score is off by d sums, its exponent (relative to the maximum, in units of log 2) by the
            # rounding of a difference of up to `reach`, the exponential itself by 2^-22: all of it
            # relative to a probability, in numerator and denominator.
            reach = np.where(np.isinf(s), 0, top - s).max(1, keepdims=True)
            delta = (d + 2) * FP32 * size.max(1, keepdims=True) + 4 * FP32 * (reach + 16) + 2.0 ** -22
            # probabilities below the type's range (fp16: multiples of 2^-24) are off by half of that;
            # the largest is at least 1
            lost = n * 2.0 ** -25 * np.abs(vh).max(0)[None] if dtype == "fp16" else 0.0
            e = u * mean + 2 * delta * mean + 2 * n * FP32 * mean + lost
            out[r, h] = o
            bound[r, h] = u * np.abs(o) * (1 + u) + e * (1 + 4 * u) + \
                (2.0 ** -25 if dtype == "fp16" else 0.0)
        at += n
    return out, bound


def rope(x, positions, freq, rotary, interleaved, amplitude, dtype):
    """x [T][heads][d] in 64 bits -> (y, bound)."""
    half = rotary // 2
    t = positions.astype(np.longdouble)[:, None] * freq.astype(np.longdouble)
    c = (np.cos(t) * amplitude).astype(np.float64)[:, None]
    s = (np.sin(t) * amplitude).astype(np.float64)[:, None]
    i = np.arange(0, rotary, 2) if interleaved else np.arange(half)
    j = i + 1 if interleaved else i + half
    y, bound = x.copy(), np.zeros(x.shape)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    # the part of a turn: three roundings of 64 bits in front, one to 32 bits behind the reduction (of up
    # to half a turn: pi * 2^-24), cos and sin to 4 units of 2^-23, the amplitude, two products, a sum
    angle = np.abs(t).astype(np.float64) * 2.0 ** -51 + np.pi * FP32 + 2.0 ** -21
    size = (np.abs(a) + np.abs(b)) * amplitude * (angle[:, None] + 4 * FP32)
    u = HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    bound[..., i] = size + u * (np.abs(y[..., i]) + size) + tiny
    bound[..., j] = size + u * (np.abs(y[..., j]) + size) + tiny
    return y, bound


def adapter(x, a, b, ranks, scales, pick, lens, base, dtype, out_dtype):
    """x [T][k], a [A][r][k], b [A][n][r], base [T][n] in 64 bits -> (out, bound)."""
    k = x.shape[1]
    out, bound = base.copy(), np.zeros(base.shape)
    u = HALF_STEP[out_dtype]
    # terms of v: half a step of the type of what the term before left (fp16: of multiples of 2^-24)
    left = {("fp16", "fp16"): 2.0 ** -21, ("fp16", "f32"): 2.0 ** -21, ("bf16", "bf16"): 2.0 ** -16,
            ("bf16", "f32"): 2.0 ** -24}[dtype, out_dtype]
    at = 0
    for n, p in zip(lens, pick):
        rows = slice(at, at + n)
        at += n
        if not 0 <= p < len(ranks):
            continue
        r = min(max(int(ranks[p]), 0), a.shape[1])
        if r == 0 or n == 0:
            continue
        ar, br = a[p, :r], b[p, :, :r]
        v = x[rows] @ ar.T
        ev = (k + 8) * FP32 * (np.abs(x[rows]) @ np.abs(ar).T)
        ev = ev + left * (np.abs(v) + ev).max(1, keepdims=True)
        y = scales[p] * (v @ br.T)
        ey = abs(scales[p]) * (ev @ np.abs(br).T + 3 * (r + 4) * FP32 * (np.abs(v) @ np.abs(br).T))
        out[rows] = base[rows] + y
        ey = ey + 2 * FP32 * (np.abs(base[rows]) + np.abs(y))
        bound[rows] = ey + u * (np.abs(out[rows]) + ey) + (2.0 ** -25 if out_dtype == "fp16" else 0)
    return out, bound


def assert_within(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (
        f"{what}: {bad.sum()} of {bad.size} outside the bound, first at "
        f"{tuple(int(i) for i in np.argwhere(bad)[0])}: {got[bad][0]} for {want[bad][0]} "
        f"+- {bound[bad][0]}")
