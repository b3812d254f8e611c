"""RMS norms of heads with rotary positions of one axis or several, against the 64-bit form."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as P
from tests import tree_reference as R

pytestmark = pytest.mark.gpu

GUARD = 2
EPS = 1e-6


def _up(a):
    return None if a is None else hip.DeviceBuffer.from_numpy(a)


def _run(rows, positions, axis, freq, gains, hq, hkv, d, rotary, dtype, interleaved=False, amplitude=1.0, eps=EPS,
         in_place=False, shift=0, stride=None):
    """rows [T][width], their first `shift` elements left out; what q_out and k_out (or the rows) hold."""
    size, (T, width) = rows.dtype.itemsize, rows.shape
    buf = hip.DeviceBuffer.from_numpy(rows)
    qi, ki = buf.offset(size * shift), buf.offset(size * (shift + hq * d)) if hkv else None
    args = [_up(a) for a in (positions, axis, freq, *gains)]
    axes = 1 if positions is None else len(positions)
    rest = dict(num_axes=axes, eps=eps, interleaved=interleaved, amplitude=amplitude, position_stride=stride,
                q_in_stride=width, k_in_stride=width, dtype=dtype)
    if in_place:
        kernels.launch_norm_rope_packed(qi, ki, qi, ki, *args, T, hq, hkv, d, rotary, q_out_stride=width,
                                        k_out_stride=width, **rest)
        hip.synchronize()
        return buf.to_numpy(rows.dtype, rows.shape)
    out = [hip.DeviceBuffer((T + GUARD) * max(h, 1) * d * size) for h in (hq, hkv)]
    for o in out:
        o.fill(0xFF)
    kernels.launch_norm_rope_packed(qi, ki, out[0], out[1] if hkv else None, *args, T, hq, hkv, d, rotary, **rest)
    hip.synchronize()
    return [o.to_numpy(rows.dtype, (T + GUARD, h * d)) for o, h in zip(out, (hq, hkv))]


def _want(x, gains, positions, axis, freq, hq, rotary, interleaved, amplitude, dtype, eps=EPS):
    parts = [R.norm_rope(x[:, s], g, eps, positions, axis, freq, rotary, interleaved, amplitude, dtype)
             for s, g in ((slice(0, hq), gains[0]), (slice(hq, None), gains[1]))]
    return [np.concatenate(p, 1).reshape(x.shape[0], -1) for p in zip(*parts)]


def _check(seed, T, hq, hkv, d, rotary, dtype, interleaved=False, axes=1, which="both", far=4000, amplitude=1.0, pad=0,
           shift=0, size=2.0, named=True):
    rng = np.random.default_rng(seed)
    heads = hq + hkv
    rows = P.to_bits(rng.standard_normal((T, shift + heads * d + pad)) * size, dtype)
    stride = T + 3 if axes > 1 else None  # (axes a little apart)
    positions = rng.integers(-far, far, (axes, T + 3 if axes > 1 else T)).astype(np.int32)
    axis = rng.integers(0, axes, rotary // 2).astype(np.uint8) if named else None
    freq = kernels.rope_frequencies(rotary, 1e4)[0] if rotary else None
    gains = [rng.uniform(0.3, 3, d).astype(np.float32) if w in which or which == "both" else None for w in "qk"]
    x = P.from_bits(rows[:, shift:shift + heads * d], dtype).reshape(T, heads, d)
    want, bound = _want(x, gains, positions[:, :T], np.zeros(rotary // 2, int) if axis is None else axis, freq, hq, rotary,
                        interleaved, amplitude, dtype)
    args = (rows, positions, axis, freq, gains, hq, hkv, d, rotary, dtype, interleaved, amplitude)
    out = _run(*args, shift=shift, stride=stride)
    for o, at in zip(out, (slice(0, hq * d), slice(hq * d, heads * d))):
        assert (o[T:].view(np.uint8) == 0xFF).all()
        P.assert_within(P.from_bits(o[:T], dtype), want[:, at], bound[:, at])
    there = _run(*args, in_place=True, shift=shift, stride=stride)
    mid = slice(shift, shift + heads * d)
    assert np.array_equal(there[:, mid], np.concatenate([o[:T] for o in out], 1))
    there[:, mid] = rows[:, mid]
    assert np.array_equal(there, rows)


DTYPES = ["fp16", "bf16", "f32"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d,rotary", [
    (14, 2, 64, 64), (12, 2, 128, 128), (4, 1, 128, 64), (2, 2, 128, 2), (3, 1, 96, 96), (2, 1, 96, 90), (5, 0, 64, 36),
    (1, 1, 2, 2), (2, 1, 34, 12), (1, 1, 256, 250), (3, 3, 7, 4), (2, 1, 512, 512), (1, 1, 1024, 1000), (2, 1, 999, 998),
    (3, 1, 80, 80), (4, 2, 256, 256)])
def test_geometries(hq, hkv, d, rotary, interleaved, dtype):
    _check(1, 1, hq, hkv, d, rotary, dtype, interleaved)
    _check(2, 37, hq, hkv, d, rotary, dtype, interleaved, axes=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "", "both"])
def test_some_heads_are_not_normed(which, dtype):
    _check(3, 11, 4, 2, 64, 64, dtype, which=which, axes=2)
    _check(4, 11, 4, 2, 128, 32, dtype, True, which=which)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 100, 257])
def test_the_norm_alone(d, dtype):
    _check(5, 9, 3, 2, d, 0, dtype)
    rng = np.random.default_rng(6)
    rows = P.to_bits(rng.standard_normal((4, 5 * d)), dtype)
    out = _run(rows, None, None, None, (None, None), 3, 2, d, 0, dtype)  # neither: copied
    assert np.array_equal(np.concatenate([o[:4] for o in out], 1), rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pad,shift", [(64, 0), (5, 0), (3, 1), (6, 2), (4, 4), (0, 8)])
def test_strides_and_addresses(pad, shift, interleaved, dtype):
    _check(7, 19, 4, 2, 64, 64, dtype, interleaved, pad=pad, shift=shift, amplitude=1.3, axes=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1023, 2050, 4097, 9000])
def test_many_tokens(T, dtype):
    _check(8, T, 2, 1, 64, 64, dtype, axes=4)
    _check(9, T, 3, 0, 64, 32, dtype, True, far=1000000, named=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_widest_rows(dtype):
    _check(10, 3, 60, 4, 1024, 1024, dtype)
    _check(11, 3, 1024, 1024, 32, 32, dtype, True)


@pytest.mark.parametrize("size", [1e-4, 1e3, 1e18, 2.0 ** 66, 1e30])
def test_small_and_large_values(size):
    """eps counts for the small ones; the squares of the large ones are beyond fp32."""
    for dtype in ("bf16", "f32"):
        _check(12, 5, 2, 1, 128, 128, dtype, size=size)
        _check(13, 5, 2, 1, 1000, 1000, dtype, size=size)
    if size < 1e4:
        _check(14, 5, 2, 1, 128, 128, "fp16", size=size)


def test_a_pair_without_an_axis_stays_at_position_0():
    rng = np.random.default_rng(15)
    T, d = 6, 64
    rows = P.to_bits(rng.standard_normal((T, 2 * d)), "f32")
    positions = rng.integers(1, 1000, (2, T)).astype(np.int32)
    axis = np.array([0, 1, 2, 255] * 8, np.uint8)
    freq = kernels.rope_frequencies(d, 1e4)[0]
    q, k = _run(rows, positions, axis, freq, (None, None), 1, 1, d, d, "f32")
    want, bound = _want(rows.astype(np.float64).reshape(T, 2, d), (None, None), positions, axis, freq, 1, d, False, 1.0, "f32")
    got = np.concatenate([q[:T], k[:T]], 1)
    P.assert_within(got, want, bound)
    still = np.concatenate([np.arange(2, 32, 4), np.arange(3, 32, 4)])
    for i in (still, still + 32, still + 64, still + 96):
        assert np.array_equal(got[:, i], rows[:, i])


def test_infinities_stay_in_their_head():
    rng = np.random.default_rng(16)
    rows = P.to_bits(rng.standard_normal((3, 6 * 64)), "f32")
    clean = rows.copy()
    rows[1, 70] = np.inf
    rows[2, 5 * 64 + 3] = np.nan
    freq = kernels.rope_frequencies(64, 1e4)[0]
    gains = [np.ones(64, np.float32)] * 2
    positions = np.array([[3, 4, 5]], np.int32)
    q, k = _run(rows, positions, None, freq, gains, 4, 2, 64, 64, "f32")
    q0, k0 = _run(clean, positions, None, freq, gains, 4, 2, 64, 64, "f32")
    got, want = np.concatenate([q, k], 1)[:3].reshape(3, 6, 64), np.concatenate([q0, k0], 1)[:3].reshape(3, 6, 64)
    assert np.isnan(got[1, 1]).any() and np.isnan(got[2, 5]).all()
    got[1, 1], got[2, 5] = want[1, 1], want[2, 5]
    assert np.array_equal(got, want)


def test_zeros_stay_zeros():
    rows = np.zeros((2, 3 * 128), np.float16)
    freq = kernels.rope_frequencies(128, 1e4)[0]
    q, k = _run(rows, np.array([[7, 8]], np.int32), None, freq, [np.ones(128, np.float32)] * 2, 2, 1, 128, 128, "fp16")
    assert not q[:2].any() and not k[:2].any()


def test_without_norm_and_with_one_axis_it_is_the_rotation():
    """Bit for bit what rotary positions alone give."""
    rng = np.random.default_rng(17)
    for dtype in DTYPES:
        T, hq, hkv, d = 50, 4, 2, 128
        rows = P.to_bits(rng.standard_normal((T, (hq + hkv) * d)), dtype)
        positions = rng.integers(0, 100000, (1, T)).astype(np.int32)
        freq = kernels.rope_frequencies(d, 1e6)[0]
        got = _run(rows, positions, None, freq, (None, None), hq, hkv, d, d, dtype, amplitude=1.1)
        buf, size = hip.DeviceBuffer.from_numpy(rows), rows.dtype.itemsize
        k = buf.offset(size * hq * d)
        w = rows.shape[1]
        kernels.launch_rope_packed(buf, k, buf, k, _up(positions[0]), _up(freq), T, hq, hkv, d, d, False, 1.1, w, w, w, w, dtype)
        hip.synchronize()
        assert np.array_equal(buf.to_numpy(rows.dtype, rows.shape), np.concatenate([g[:T] for g in got], 1))
