"""Operators over packed rows where what carries the result is far smaller than what lies beside it, or
far larger than a type's ordinary values: against 64-bit forms, within the bounds that the documented
roundings add up to."""
import numpy as np
import pytest

from tests import packed_reference as R
from tests import test_gpu_adapter_add as D
from tests import test_gpu_attn_packed as A

pytestmark = pytest.mark.gpu

FAR = [  # lengths, query and KV heads, head width
    ([1, 33, 150], 4, 2, 64), ([70, 200], 4, 2, 256), ([1090], 4, 2, 64), ([1090], 4, 2, 128),
    ([4097, 4200], 24, 8, 128)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,hq,hkv,d", FAR)
def test_scores_that_are_finite_before_the_scale_only(lens, hq, hkv, d, dtype, causal):
    """All scores of a sequence times the scale lie below what fp32 holds, and their differences are finite (and huge):
    a row is the mean of v over its best keys."""
    one, low, scale = (2.0 ** 8, 2.0 ** 8, 2.0 ** 114) if dtype == "fp16" else (2.0 ** 63, 2.0 ** 62, 16.0)
    rng = np.random.default_rng(3)
    T, n_all = sum(lens) + A.GUARD, sum(lens)
    q, k = np.zeros((T, hq, d)), np.zeros((T, hkv, d))
    q[..., 0] = one
    level = rng.integers(1, 4, T)
    k[..., 0] = -low * level[:, None]  # (times `one` and the scale: at most -2^129)
    v = rng.integers(-8, 9, (T, hkv, d)).astype(np.float64)
    rows = np.concatenate([x.reshape(T, -1) for x in (q, k, v)], 1)
    c = dict(rows=R.to_bits(rows, dtype), lens=lens, hq=hq, hkv=hkv, d=d, dtype=dtype, fused=False, T=T)
    assert (R.from_bits(c["rows"], dtype) == rows).all()
    r = A.Run(c, causal, scale)
    r.launch()
    got = r.result().reshape(n_all, hq, d)
    at = 0
    for n in lens:
        here = level[at:at + n]
        best = np.minimum.accumulate(here) if causal else np.full(n, here.min())
        for h in range(hq):
            vh = v[at:at + n, h // (hq // hkv)]
            want = np.zeros((n, d))
            for b in (1, 2, 3):
                mine = here == b
                if causal:
                    mean = np.cumsum(vh * mine[:, None], 0) / np.maximum(np.cumsum(mine), 1)[:, None]
                else:
                    mean = np.broadcast_to((vh * mine[:, None]).sum(0) / max(mine.sum(), 1), (n, d))
                want[best == b] = mean[best == b]
            # the result's rounding, the reciprocal's and the product's in fp32; sums of ones and integers are exact
            u = R.HALF_STEP[dtype]
            R.assert_within(got[at:at + n, h], want, (u * (1 + 2.0 ** -20) + 3 * R.FP32) * np.abs(want)
                            + (2.0 ** -25 if dtype == "fp16" else 0.0), f"sequence of {n}, head {h}")
        at += n


HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
SCALE = float(np.float32(np.log(2)))  # scores are powers of two then


def _attn_case(lens, hq, hkv, d, dtype, scores, v, odd_head):
    """Queries (1, 0, ..): the score of a key is its first element.  odd_head: the last query head of
    every group is NaN, so that every workgroup goes through its keys a second time."""
    T = sum(lens) + A.GUARD
    q, k = np.zeros((T, hq, d)), np.zeros((T, hkv, d))
    q[..., 0] = 1.0
    k[:len(scores), :, 0] = scores[:, None]
    rows = R.to_bits(np.concatenate([x.reshape(T, -1) for x in (q, k, v)], 1), dtype)
    assert np.array_equal(R.from_bits(rows[:, hq * d:(hq + hkv) * d:d], dtype), k[..., 0])
    if odd_head:
        g = hq // hkv
        rows[:, :hq * d].reshape(T, hkv, g, d)[:, :, g - 1] = A._nan(dtype)
    return dict(rows=rows, lens=lens, hq=hq, hkv=hkv, d=d, dtype=dtype, fused=False, T=T)


FORMS = [  # lengths, query and KV heads, head width
    ([300], 2, 1, 64), ([4096], 2, 1, 192), ([4096], 2, 1, 64), ([4096], 2, 1, 128),
    ([4097, 4200], 24, 8, 128), ([16384], 4, 2, 64)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("odd_head", [False, True], ids=["", "second walk"])
@pytest.mark.parametrize("below", [16.0, 18.625, 21.5, 23.5, 25.25])
@pytest.mark.parametrize("lens,hq,hkv,d", FORMS)
def test_many_small_weights_beside_one_of_nothing(lens, hq, hkv, d, below, odd_head, dtype):
    """One key of each sequence outweighs every other one by 2^below and has a V row of zeros: the result
    is what the others add up to."""
    rng = np.random.default_rng(1)
    T, n_all = sum(lens) + A.GUARD, sum(lens)
    v = np.broadcast_to(1.0 + rng.integers(0, 8, (hkv, d)) / 8, (T, hkv, d)).copy()
    scores = np.full(n_all, -below)
    at = 0
    sinks = []
    for i, n in enumerate(lens):
        sinks.append(at + (0 if i % 2 == 0 else n // 2))
        at += n
    scores[sinks] = 0.0
    v[sinks] = 0.0
    c = _attn_case(lens, hq, hkv, d, dtype, scores, v, odd_head)
    g, u = hq // hkv, HALF[dtype]
    heads = [h for h in range(hq) if not (odd_head and h % g == g - 1)]
    w = np.exp(-below * SCALE)
    # A weight is rounded to the rows' type (fp16: those below 2^-25 of the largest to multiples of 2^-35 of
    # it); its exponent is a rounded difference, the exponential good to 2^-22.
    one = max(u * w, 2.0 ** -36 if dtype == "fp16" else 0.0)
    delta = 4 * R.FP32 * (below + 16) + 2.0 ** -22
    for causal in (False, True):
        r = A.Run(c, causal, SCALE)
        r.launch()
        got = r.result().reshape(n_all, hq, d)
        at = 0
        for n, sink in zip(lens, sinks):
            t = np.arange(n)
            seen = t + 1.0 if causal else np.full(n, float(n))
            there = (t >= sink - at) if causal else np.ones(n, bool)  # sees the heavy key
            others = seen - there
            weight = np.where(there, w, 1.0)
            total = others * weight + there
            mean = (others * weight / total)[:, None]
            lost = (others * np.where(there, one, u) / total)[:, None]
            for h in heads:
                value = v[at + (1 if sink == at else 0), h // g][None]
                o = mean * value
                e = lost * value + (2 * delta + 2 * n * R.FP32) * o
                bound = u * o * (1 + u) + e * (1 + 4 * u) + (2.0 ** -25 if dtype == "fp16" else 0.0)
                R.assert_within(got[at:at + n, h], o, bound, f"causal={causal}, sequence of {n}, head {h}")
            at += n
        if odd_head:
            assert np.isnan(got[:, g - 1]).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_weights_that_only_count_together(dtype):
    """131072 keys, each 2^-25.25 of the first, whose V row is zero."""
    n, d, below = 131072, 64, 25.25
    v = np.full((n + A.GUARD, 1, d), 1.5)
    v[0] = 0.0
    scores = np.full(n, -below)
    scores[0] = 0.0
    c = _attn_case([n], 1, 1, d, dtype, scores, v, False)
    r = A.Run(c, False, SCALE)
    r.launch()
    got, w, u = r.result(), np.exp(-below * SCALE), HALF[dtype]
    total = 1 + (n - 1) * w
    o = (n - 1) * w / total * 1.5
    one = max(u * w, 2.0 ** -36 if dtype == "fp16" else 0.0)
    e = (n - 1) * one / total * 1.5 + (2 * (4 * R.FP32 * (below + 16) + 2.0 ** -22) + 2 * n * R.FP32) * o
    R.assert_within(got, np.full_like(got, o), u * o * (1 + u) + e * (1 + 4 * u) + 2.0 ** -25)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("step", [1, 4, 8])
def test_scores_that_rise_little_by_little(step, d, dtype):
    """From key to key by step eighths of a power of two: what the weights are relative to lies as far below
    the largest as it may, and the largest as high in the type."""
    n = 256 // step
    rng = np.random.default_rng(2)
    v = rng.integers(1, 9, (n + 2 * n + A.GUARD, 2, d)) / 4.0
    scores = np.concatenate([np.arange(n) * step, np.repeat(np.arange(n), 2) * step // 2]) / 8.0
    lens = [n, 2 * n]
    c = _attn_case(lens, 4, 2, d, dtype, np.floor(scores * 8) / 8, v, False)
    for causal in (False, True):
        A._check(c, causal, SCALE)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("odd_head", [False, True], ids=["", "second walk"])
@pytest.mark.parametrize("lens,hq,hkv,d", [([2, 33, 150], 4, 2, 64), ([70, 200], 4, 2, 256), ([1090], 4, 2, 64),
                                           ([1090], 4, 2, 128), ([4097, 4200], 24, 8, 128)])
def test_the_mean_of_the_largest_values(lens, hq, hkv, d, odd_head, causal):
    """bf16 values up to 2^127, of which two add up to more than fp32 holds: their weighted mean is finite."""
    rng = np.random.default_rng(4)
    c = A._case(23, lens, hq, hkv, d, "bf16")
    q, _, v = A._parts(c)
    v[:] = R.to_bits(rng.uniform(0.5, 1, v.shape) * 2.0 ** 127, "bf16")
    n, g, kvh = sum(lens), hq // hkv, hkv - 1
    heads = np.arange(kvh * g, kvh * g + g - odd_head)  # (those of the last KV head, the odd ones left out)
    bits = [np.ascontiguousarray(x[:n]) for x in A._parts(c)]
    if odd_head:
        q.reshape(len(q), hkv, g, d)[:, :, g - 1] = A._nan("bf16")
    r = A.Run(c, causal)
    r.launch()
    got = r.result().reshape(n, hq, d)
    fq, fk, fv = (R.from_bits(x, "bf16").reshape(n, -1, d) for x in bits)
    want, bound = R.attention(fq[:, heads], fk[:, kvh:kvh + 1], fv[:, kvh:kvh + 1], lens, r.scale, causal, "bf16")
    R.assert_within(got[:, heads], want, bound)


# What the terms of x . A^T are off by: relative to the value itself, and to the largest of its row.
TERMS = {("fp16", "fp16"): (2.0 ** -22, 2.0 ** -39), ("bf16", "bf16"): (2.0 ** -16, 0.0),
         ("fp16", "f32"): (2.0 ** -33, 2.0 ** -39), ("bf16", "f32"): (2.0 ** -24, 0.0)}
TILES = [[1, 16, 3], [40, 1, 90], [1, 2] * 150, [33] * 40]


def _uneven_case(lens, max_rank, n, below, dtype, out):
    """The first rank's value is 2^below times the others' and its column of B zero: x holds a large and a small
    element, A one of them per rank."""
    k = 128
    c = D._case(24, lens, np.arange(len(lens)) % 2, [max_rank, max_rank - 3], max_rank, n, k, dtype, out)
    rng = np.random.default_rng(5)

    def between(*shape):
        return rng.uniform(1, 2, shape) * rng.choice([-1, 1], shape)

    x, a = np.zeros(c["x"].shape), np.zeros(c["a"].shape)
    x[:, 40], x[:, 7] = 2.0 ** 10 * between(len(x)), between(len(x))
    a[:, 0, 40], a[:, 1:, 7] = 2.0 ** 10 * between(2), 2.0 ** (20 - below) * between(2, max_rank - 1)
    b = R.from_bits(c["b"], dtype)
    b[:, :, 0] = 0.0
    c["x"], c["a"], c["b"] = (R.to_bits(y, dtype) for y in (x, a, b))
    c["base"] = np.zeros_like(c["base"])
    return c


def _uneven_want(c, terms):
    f = lambda y: R.from_bits(y, c["dtype"])  # noqa: E731
    n, u = sum(c["lens"]), R.HALF_STEP[c["out_dtype"]]
    want, bound, at = np.zeros((n, c["n"])), np.zeros((n, c["n"])), 0
    for i, p in zip(c["lens"], c["pick"]):
        r, s = c["ranks"][p], float(c["scales"][p])
        v = f(c["x"][at:at + i]) @ f(c["a"][p, :r]).T * s
        b = f(c["b"][p, :, :r]).T
        # v: one product that counts, its sum and the scale in fp32; then its terms and the sum over the ranks
        e = np.abs(v) * (4 * R.FP32 + terms[0]) + np.abs(v).max(1, keepdims=True) * terms[1]
        y = v @ b
        ey = e @ np.abs(b) + 3 * (r + 4) * R.FP32 * (np.abs(v) @ np.abs(b))
        want[at:at + i], bound[at:at + i] = y, ey + u * (np.abs(y) + ey) + (
            2.0 ** -25 if c["out_dtype"] == "fp16" else 0.0)
        at += i
    return want, bound


@pytest.mark.parametrize("dtype,out", list(TERMS))
@pytest.mark.parametrize("below", [12, 18, 22, 26])
@pytest.mark.parametrize("max_rank", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens", TILES, ids=lambda v: f"{len(v)} of {max(v)}")
def test_small_ranks_beside_a_large_one(lens, max_rank, below, dtype, out):
    c = _uneven_case(lens, max_rank, 264, below, dtype, out)
    r = D.Run(c)
    r.launch()
    R.assert_within(R.from_bits(r.bits()[:sum(lens)], out), *_uneven_want(c, TERMS[dtype, out]))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("max_rank", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens", TILES, ids=lambda v: f"{len(v)} of {max(v)}")
def test_fp32_results_have_all_bits_of_the_first_product(lens, max_rank, dtype):
    """x . A^T has 24 bits, every row of B one power of two: the results are exact."""
    c = D._case(25, lens, np.arange(len(lens)) % 2, [max_rank, max_rank - 3], max_rank, 264, 128, dtype, "f32")
    rng = np.random.default_rng(6)
    bits, step = (11, 2.0 ** -2) if dtype == "fp16" else (8, 2.0 ** -8)

    def odd(lo, hi, *shape):
        return 2.0 * rng.integers(lo // 2, hi // 2, shape) + 1

    x, a, b = np.zeros(c["x"].shape), np.zeros(c["a"].shape), np.zeros(c["b"].shape)
    x[:, 40], a[:, :, 40] = odd(1 << bits - 1, 1 << bits, len(x)), odd(1 << bits - 1, 1 << bits, 2, max_rank)
    # (added a step of 32 columns earlier: 22 or 16 bits in front of the point, 2 or 8 behind it)
    x[:, 7], a[:, :, 7] = 1.0, odd(0, round(1 / step), 2, max_rank) * step
    b[:, np.arange(264), np.arange(264) % (max_rank - 3)] = 2.0 ** rng.integers(-4, 5, (2, 264))
    c["x"], c["a"], c["b"] = (R.to_bits(y, dtype) for y in (x, a, b))
    for bits_of, y in zip((c["x"], c["a"], c["b"]), (x, a, b)):
        assert (R.from_bits(bits_of, dtype) == y).all()
    c["base"], c["scales"] = np.zeros_like(c["base"]), np.array([1.0, 2.0], np.float32)
    r = D.Run(c)
    r.launch()
    got, at = r.bits(), 0
    for n, p in zip(c["lens"], c["pick"]):
        want = (x[at:at + n] @ a[p].T) @ b[p].T * (1 + p)
        assert (want == want.astype(np.float32)).all()
        assert np.array_equal(got[at:at + n], want.astype(np.float32))
        at += n


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("max_rank", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens", TILES, ids=lambda v: f"{len(v)} of {max(v)}")
def test_sums_that_pass_the_range_only_before_they_are_scaled(lens, max_rank, out):
    """bf16 rows near 2^-60 and B near 2^127: a sum over the ranks of B alone is more than fp32 holds."""
    c = D._case(26, lens, np.arange(len(lens)) % 2, [max_rank, max_rank - 3], max_rank, 264, 128, "bf16", out)
    rng = np.random.default_rng(7)
    c["x"] = R.to_bits(rng.uniform(0.5, 1, c["x"].shape) * 2.0 ** -60, "bf16")
    c["a"] = R.to_bits(rng.uniform(0.5, 1, c["a"].shape), "bf16")
    c["b"] = R.to_bits(rng.uniform(0.5, 1, c["b"].shape) * 2.0 ** 127, "bf16")
    r = D.Run(c)
    r.launch()
    R.assert_within(R.from_bits(r.bits()[:sum(lens)], out), *D._want(c))
