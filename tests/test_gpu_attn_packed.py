"""Attention of whole packed sequences against the 64-bit form, element by element within the bound
that the documented roundings add up to."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as R

pytestmark = pytest.mark.gpu

GUARD = 3  # rows behind the last sequence


def _case(seed, lens, hq, hkv, d, dtype, fused=False, size=1.0):
    rng = np.random.default_rng(seed)
    T = int(sum(lens)) + GUARD
    width = (hq + 2 * hkv) * d
    rows = R.to_bits(rng.standard_normal((T, width), np.float32) * np.float32(size), dtype)
    return dict(rows=rows, lens=list(lens), hq=hq, hkv=hkv, d=d, dtype=dtype, fused=fused, T=T)


def _parts(c):
    a, b = c["hq"] * c["d"], c["hkv"] * c["d"]
    r = c["rows"]
    return r[:, :a], r[:, a:a + b], r[:, a + b:]


class Run:
    def __init__(self, c, causal, scale=None, stream=None, out_pad=0):
        self.c, self.causal, self.stream = c, causal, stream
        self.scale = scale or 1.0 / np.sqrt(c["d"])
        q, k, v = _parts(c)
        self.qw, self.out_stride = q.shape[1], q.shape[1] + out_pad
        if c["fused"]:
            self.rows = hip.DeviceBuffer.from_numpy(c["rows"])
            at = [self.rows.offset(2 * x) for x in (0, q.shape[1], q.shape[1] + k.shape[1])]
            self.strides = [c["rows"].shape[1]] * 3
        else:
            self.rows = [hip.DeviceBuffer.from_numpy(x) for x in (q, k, v)]
            at, self.strides = self.rows, [q.shape[1], k.shape[1], v.shape[1]]
        self.at = at
        self.cu = hip.DeviceBuffer.from_numpy(np.concatenate([[0], np.cumsum(c["lens"])]).astype(np.int32))
        self.out = hip.DeviceBuffer(c["T"] * self.out_stride * 2)
        self.out.fill(0xFF)

    def launch(self):
        c = self.c
        kernels.launch_attn_packed(*self.at, self.cu, self.out, len(c["lens"]), c["T"], c["hq"],
                                   c["hkv"], c["d"], self.scale, self.causal, *self.strides,
                                   self.out_stride, bf16=c["dtype"] == "bf16", stream=self.stream)

    def bits(self):
        (self.stream.synchronize() if self.stream else hip.synchronize())
        return self.out.to_numpy(np.uint16, (self.c["T"], self.out_stride))

    def result(self):
        """The rows of the sequences in 64 bits; what lies behind and beside them is as it was."""
        got = self.bits()
        n = sum(self.c["lens"])
        assert (got[n:] == 0xFFFF).all() and (got[:, self.qw:] == 0xFFFF).all()
        got = got[:n, :self.qw]
        got = got.view(np.float16) if self.c["dtype"] == "fp16" else got
        return R.from_bits(np.ascontiguousarray(got), self.c["dtype"])


def _want(c, causal, scale=None):
    n = sum(c["lens"])
    q, k, v = (R.from_bits(np.ascontiguousarray(x[:n]), c["dtype"]).reshape(n, -1, c["d"])
               for x in _parts(c))
    o, bound = R.attention(q, k, v, c["lens"], scale or 1.0 / np.sqrt(c["d"]), causal, c["dtype"])
    return o.reshape(n, -1), bound.reshape(n, -1)


def _check(c, causal, scale=None, **kw):
    r = Run(c, causal, scale, **kw)
    r.launch()
    R.assert_within(r.result(), *_want(c, causal, scale),
                    what=f"{c['lens']} {c['hq']}/{c['hkv']} x {c['d']} {c['dtype']} causal={causal}")
    return r


LENGTHS = [[1], [2, 1, 1], [1, 0, 5, 33], [31, 32, 33, 64, 65], [0, 0, 7, 0], [127, 128, 129],
           [300, 1, 17]]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (14, 2, 64), (12, 2, 128), (8, 1, 128)])
def test_lengths(lens, hq, hkv, d, causal, dtype):
    _check(_case(1, lens, hq, hkv, d, dtype), causal)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
def test_widths(d, causal, dtype):
    _check(_case(2, [70, 3, 200, 40], 6, 2, d, dtype), causal)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (9, 3), (32, 1), (40, 1), (7, 7), (48, 16)])
@pytest.mark.parametrize("d", [64, 128])
def test_groups(hq, hkv, d):
    _check(_case(3, [1, 50, 97], hq, hkv, d, "fp16"), True)
    _check(_case(4, [1, 50, 97], hq, hkv, d, "bf16"), False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128), (4, 2, 96), (4, 2, 256)])
def test_columns_of_fused_rows(hq, hkv, d, dtype):
    c = _case(5, [129, 1, 64, 31], hq, hkv, d, dtype, fused=True)
    _check(c, True, out_pad=8)
    _check(c, False)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_many_key_tiles(d, causal, dtype):
    _check(_case(6, [1500, 777], 2, 1, d, dtype), causal)


@pytest.mark.parametrize("hq,hkv,d,lens", [(16, 2, 128, [900, 1100, 650]), (16, 4, 64, [2100, 333]),
                                           (8, 1, 128, [2600]), (16, 16, 64, [600] * 3)])
def test_many_workgroups(hq, hkv, d, lens):
    _check(_case(16, lens, hq, hkv, d, "bf16", fused=True), True)


def test_many_short_sequences():
    rng = np.random.default_rng(7)
    _check(_case(7, rng.integers(0, 5, 700), 4, 2, 64, "bf16"), True)
    _check(_case(8, rng.integers(0, 40, 130), 4, 2, 128, "fp16"), False)


@pytest.mark.parametrize("d", [64, 128, 192])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_large_scores(d, dtype):
    """Scores up to some hundreds: the running maximum rises by much, often and late."""
    c = _case(9, [260, 90], 4, 2, d, dtype, size=4.0)
    _check(c, True)
    # rising and falling along the keys
    q, k, _ = _parts(c)
    order = np.linspace(0.05, 3.0, c["T"])[:, None]
    k[:] = R.to_bits(R.from_bits(np.ascontiguousarray(k), dtype) * order, dtype)
    _check(c, False)
    k[:] = k[::-1].copy()
    _check(c, True)


@pytest.mark.parametrize("scale", [1e-4, 1.0])
def test_scales(scale):
    _check(_case(10, [100, 60], 4, 2, 128, "fp16"), True, scale)
    _check(_case(10, [100, 60], 4, 2, 64, "bf16"), False, scale)


def _nan(dtype):
    return np.float16(np.nan) if dtype == "fp16" else np.uint16(0x7FC0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("n,bad", [(70, 33), (70, 69), (40, 1), (300, 200), (300, 129)])
def test_what_later_keys_hold_does_not_reach_a_token(d, n, bad, dtype):
    """NaN in the K and V rows of token `bad` and in everything of the sequence behind: tokens in
    front of it keep their results, those that see it are NaN."""
    c = _case(11, [n, 50], 6, 2, d, dtype)
    want, bound = _want(c, True)
    q, k, v = _parts(c)
    q, k, v = q.copy(), k.copy(), v.copy()
    k[bad], v[bad] = _nan(dtype), _nan(dtype)
    k[n:n + 50], v[n:n + 50], q[n:n + 50] = _nan(dtype), _nan(dtype), _nan(dtype)
    c["rows"] = np.concatenate([q, k, v], 1)
    r = Run(c, True)
    r.launch()
    got = r.result()
    R.assert_within(got[:bad], want[:bad], bound[:bad])
    assert np.isnan(got[bad:]).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_infinite_values_of_later_keys(d, dtype):
    c = _case(12, [90], 4, 4, d, dtype)
    want, bound = _want(c, True)
    _, _, v = _parts(c)
    v[45] = np.float16(np.inf) if dtype == "fp16" else np.uint16(0x7F80)
    r = Run(c, True)
    r.launch()
    got = r.result()
    R.assert_within(got[:45], want[:45], bound[:45])
    assert np.isposinf(got[45:]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_keys_that_all_score_minus_infinity_give_zeros(d):
    c = _case(13, [40, 3], 2, 2, d, "bf16")
    q, k, _ = _parts(c)
    q[:] = np.uint16(0x3F80)  # 1
    k[:5] = np.uint16(0xFF80)  # -inf
    r = Run(c, True)
    r.launch()
    got = r.result()
    assert (got[:5] == 0).all() and np.isfinite(got).all()


@pytest.mark.parametrize("d", [64, 128])
def test_lengths_past_the_rows_are_cut(d):
    """cu_seqlens that names more rows than there are: those that are there count."""
    c = _case(14, [20, 30], 4, 2, d, "fp16")
    r = Run(c, True)
    cu = np.array([0, 20, 5000], np.int32)
    r.cu.copy_from_host(cu)
    r.launch()
    c2 = dict(c, lens=[20, 30 + GUARD])
    got = R.from_bits(r.bits().view(np.float16), "fp16")
    R.assert_within(got, *_want(c2, True))


def test_a_captured_call_replays():
    stream = hip.Stream()
    c = _case(15, [129, 40, 1], 4, 2, 128, "bf16")
    r = Run(c, True, stream=stream)
    r.launch()
    want = r.bits().copy()
    r.out.fill(0xFF)
    hip.synchronize()
    graph = hip.Graph(stream)
    with graph:
        r.launch()
    for _ in range(3):
        r.out.fill(0xFF)
        hip.synchronize()
        graph.launch()
        assert np.array_equal(r.bits(), want)
        r.launch()
        assert np.array_equal(r.bits(), want)


def test_two_streams_at_once():
    runs = [Run(_case(20 + i, [200 + i, 77], 8, 2, 64, "fp16"), True, stream=hip.Stream())
            for i in range(2)]
    for _ in range(4):
        for r in runs:
            r.launch()
    for r in runs:
        R.assert_within(r.result(), *_want(r.c, True))


@pytest.mark.parametrize("negative", [False, True])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_scores_of_which_fp32_holds_no_fraction(dtype, d, causal, negative):
    """Scores of 2^31 and more: half a step of such a number is hundreds of powers of two, so what a
    product and its rounded value differ by must not get into an exponent."""
    rng = np.random.default_rng(d + negative)
    lens, hq, hkv, scale = [1, 33, 150], 4, 2, 4.0
    T = sum(lens) + GUARD
    # small integers times powers of two: every sum is exact in fp32, equal scores are equal, and different ones at
    # least 2^27 apart, so a row is the mean of v over its best keys
    q = 2.0 ** 13 * (np.ones((T, hq, d)) if negative else rng.choice([-1.0, 1.0], (T, hq, d)))
    k = 2.0 ** 12 * (-rng.integers(1, 9, (T, hkv, d)) if negative else rng.integers(-8, 9, (T, hkv, d)))
    v = rng.integers(-8, 9, (T, hkv, d)).astype(np.float64)
    rows = np.concatenate([x.reshape(T, -1) for x in (q, k, v)], 1)
    c = dict(rows=R.to_bits(rows, dtype), lens=lens, hq=hq, hkv=hkv, d=d, dtype=dtype, fused=False, T=T)
    assert (R.from_bits(c["rows"], dtype) == rows).all()
    run = Run(c, causal, scale)
    run.launch()
    got = run.result().reshape(-1, hq, d)
    at = 0
    for n in lens:
        r = slice(at, at + n)
        for h in range(hq):
            s = (q[r, h] @ k[r, h // 2].T) * scale
            if causal:
                s[np.triu(np.ones((n, n), bool), 1)] = -np.inf
            best = (s == s.max(1, keepdims=True)).astype(np.float64)
            want = best @ v[r, h // 2] / best.sum(1, keepdims=True)
            # the result's rounding, the reciprocal's and the product's in fp32; sums of ones and integers are exact
            bound = R.HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -20) + 3 * R.FP32 * np.abs(want)
            R.assert_within(got[r, h], want, bound, f"sequence of {n}, head {h}")
        at += n


@pytest.mark.parametrize("dtype,causal", [("bf16", True), ("fp16", False)])
def test_long_sequences_with_heads_of_128(dtype, causal):
    """Sequences and heads enough for the form with 256 columns to a workgroup: its results, and with a
    token whose K and V rows are NaN those of the tokens in front of it and of the other sequence."""
    hq, hkv, d, lens, kvh, bad = 24, 8, 128, [4097, 4200], 5, 2000
    c = _case(17, lens, hq, hkv, d, dtype)
    r = Run(c, causal)
    r.launch()
    clean = r.bits().copy()
    n, heads = sum(lens), slice(3 * kvh, 3 * kvh + 3)
    q, k, v = (R.from_bits(np.ascontiguousarray(x[:n]), dtype).reshape(n, -1, d) for x in _parts(c))
    want, bound = R.attention(q[:, heads], k[:, kvh:kvh + 1], v[:, kvh:kvh + 1], lens, r.scale, causal, dtype)
    R.assert_within(r.result().reshape(n, hq, d)[:, heads], want, bound)

    _, k, v = _parts(c)
    k[bad], v[bad] = _nan(dtype), _nan(dtype)
    r = Run(c, causal)
    r.launch()
    got = r.result()
    first = bad if causal else 0
    assert np.isnan(got[first:lens[0]]).all()
    assert np.array_equal(r.bits()[lens[0]:], clean[lens[0]:])
    R.assert_within(got.reshape(n, hq, d)[:first, heads], want[:first], bound[:first])


def test_long_sequences_with_scores_beyond_the_fraction():
    """The same form with one key of each sequence far above all others: its row of v is the result."""
    hq, hkv, d, lens, dtype = 24, 8, 128, [4097, 4200], "bf16"
    c = _case(18, lens, hq, hkv, d, dtype)
    q, k, v = _parts(c)
    q[:] = R.to_bits(np.full((1,), 2.0 ** 14), dtype)
    k[:] = R.to_bits(np.full((1,), -2.0 ** 12), dtype)
    best, at = [70, 4097 + 4000], 0  # (the weight of all others is 2^-(2^29) and less)
    k[best] = R.to_bits(np.full((1,), -2.0 ** 11), dtype)
    r = Run(c, True)
    r.launch()
    got = r.result().reshape(-1, hq, d)
    vals = R.from_bits(np.ascontiguousarray(v), dtype).reshape(-1, hkv, d)
    for n, b in zip(lens, best):
        for h in range(hq):
            want = np.broadcast_to(vals[b, h // 3], (at + n - b, d))
            assert np.array_equal(got[b:at + n, h], want)
        assert np.isfinite(got[at:b]).all()
        at += n


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[1056], [3100, 1, 33], [0, 2113, 31]], ids=str)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_few_long_sequences(d, lens, causal, dtype):
    """Key tiles dealt out to two parts of a workgroup: odd numbers of tiles, sequences and columns of which the
    second part sees no key."""
    _check(_case(19, lens, 4, 2, d, dtype, fused=True), causal)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("bad", [1, 33, 640, 1089])
def test_later_keys_of_few_long_sequences(d, bad, dtype):
    c = _case(20, [1090], 4, 2, d, dtype)
    want, bound = _want(c, True)
    q, k, v = _parts(c)
    k[bad], v[bad] = _nan(dtype), _nan(dtype)
    r = Run(c, True)
    r.launch()
    got = r.result()
    R.assert_within(got[:bad], want[:bad], bound[:bad])
    assert np.isnan(got[bad:]).all()


@pytest.mark.parametrize("negative", [False, True])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_scores_beyond_the_fraction_of_few_long_sequences(d, negative):
    """One key far above the others (all scores below zero, or above it): its row of v, wherever it lies."""
    n, hq, hkv, dtype = 1090, 4, 2, "bf16"
    for best in (0, 31, 32, 700, 1089):
        c = _case(21, [n], hq, hkv, d, dtype)
        q, k, v = _parts(c)
        q[:] = R.to_bits(np.full((1,), 2.0 ** 14), dtype)
        low, high = (-2.0 ** 12, -2.0 ** 11) if negative else (2.0 ** 11, 2.0 ** 12)
        k[:] = R.to_bits(np.full((1,), low), dtype)
        k[best] = R.to_bits(np.full((1,), high), dtype)
        r = Run(c, True, scale=16.0)
        r.launch()
        got = r.result().reshape(n, hq, d)
        vals = R.from_bits(np.ascontiguousarray(v), dtype).reshape(n + GUARD, hkv, d)
        for h in range(hq):
            assert np.array_equal(got[best:, h], np.broadcast_to(vals[best, h // 2], (n - best, d)))
        assert np.isfinite(got).all()


@pytest.mark.parametrize("d", [64, 128])
def test_keys_of_few_long_sequences_that_score_minus_infinity(d):
    """The first token sees only such keys, then one part of the workgroup does: zeros, and the mean over the rest."""
    c = _case(22, [1090], 2, 2, d, "bf16")
    q, k, v = _parts(c)
    q[:], k[:] = np.uint16(0x3F80), np.uint16(0)  # 1; 0: all that count score the same
    hidden = np.arange(1090 + GUARD) // 32 % 2 == 0
    k[hidden] = np.uint16(0xFF80)  # -inf
    r = Run(c, True)
    r.launch()
    got = r.result()
    assert (got[:32] == 0).all()
    seen = np.where(hidden[:1090, None], 0.0, R.from_bits(np.ascontiguousarray(v[:1090]), "bf16"))
    count = np.maximum(np.cumsum(~hidden[:1090]), 1)[:, None]
    want, size = np.cumsum(seen, 0) / count, np.cumsum(np.abs(seen), 0) / count
    # probabilities are exact ones; sums of up to 1090 terms, the reciprocal, the product, the result's rounding
    R.assert_within(got, want, R.HALF_STEP["bf16"] * np.abs(want) * (1 + 2.0 ** -7) + 1100 * R.FP32 * size)
