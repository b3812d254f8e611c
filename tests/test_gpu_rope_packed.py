"""Rotary positions of packed rows against the 64-bit form."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as R

pytestmark = pytest.mark.gpu

GUARD = 2


def _launch(rows_bits, positions, freq, hq, hkv, d, rotary, dtype, interleaved=False, amplitude=1.0,
            in_place=False, pad=0, shift=0, stream=None):
    """rows [T][(hq + hkv) * d + pad], their first `shift` elements left out; returns what q_out and
    k_out hold, guard rows included."""
    size = rows_bits.dtype.itemsize
    T = len(positions)
    width = rows_bits.shape[1]
    rows = hip.DeviceBuffer.from_numpy(rows_bits)
    qi, ki = rows.offset(size * shift), rows.offset(size * (shift + hq * d))
    pos, f = hip.DeviceBuffer.from_numpy(positions), hip.DeviceBuffer.from_numpy(freq)
    if in_place:
        kernels.launch_rope_packed(qi, ki if hkv else None, qi, ki if hkv else None, pos, f, T, hq,
                                   hkv, d, rotary, interleaved, amplitude, width, width, width, width,
                                   dtype, stream)
        hip.synchronize()
        return rows.to_numpy(rows_bits.dtype, rows_bits.shape)
    out = [hip.DeviceBuffer((T + GUARD) * max(h, 1) * d * size) for h in (hq, hkv)]
    for o in out:
        o.fill(0xFF)
    kernels.launch_rope_packed(qi, ki if hkv else None, out[0], out[1] if hkv else None, pos, f, T, hq,
                               hkv, d, rotary, interleaved, amplitude, width, width, dtype=dtype,
                               stream=stream)
    hip.synchronize()
    return [o.to_numpy(rows_bits.dtype, (T + GUARD, h * d)) for o, h in zip(out, (hq, hkv))]


def _rows(rng, T, width, dtype):
    return R.to_bits(rng.standard_normal((T, width), np.float32), dtype)


def _check(seed, T, hq, hkv, d, rotary, dtype, interleaved, far=4000, amplitude=1.0, pad=0, shift=0,
           positions=None):
    rng = np.random.default_rng(seed)
    rows = _rows(rng, T, shift + (hq + hkv) * d + pad, dtype)
    if positions is None:
        positions = rng.integers(0, far, T).astype(np.int32)
    freq, _ = kernels.rope_frequencies(rotary, 1e4)
    x = R.from_bits(rows[:, shift:shift + (hq + hkv) * d], dtype).reshape(T, hq + hkv, d)
    want, bound = R.rope(x, positions, freq, rotary, interleaved, amplitude, dtype)
    want, bound = want.reshape(T, -1), bound.reshape(T, -1)
    out = _launch(rows, positions, freq, hq, hkv, d, rotary, dtype, interleaved, amplitude, pad=pad,
                  shift=shift)
    for o, at in zip(out, (slice(0, hq * d), slice(hq * d, (hq + hkv) * d))):
        assert (o[T:].view(np.uint8) == 0xFF).all()  # rows behind the last are as they were
        R.assert_within(R.from_bits(o[:T], dtype), want[:, at], bound[:, at])
    # in place: the same bits, and nothing else of the rows changes
    there = _launch(rows, positions, freq, hq, hkv, d, rotary, dtype, interleaved, amplitude, True,
                    pad=pad, shift=shift)
    both = np.concatenate([o[:T] for o in out], 1)
    mid = slice(shift, shift + (hq + hkv) * d)
    assert np.array_equal(there[:, mid], both)
    there[:, mid] = rows[:, mid]
    assert np.array_equal(there, rows)


DTYPES = ["fp16", "bf16", "f32"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d,rotary", [
    (14, 2, 64, 64), (12, 2, 128, 128), (4, 1, 128, 64), (2, 2, 128, 2), (3, 1, 96, 96), (2, 1, 96, 90),
    (5, 0, 64, 36), (1, 1, 2, 2), (2, 1, 34, 12), (1, 1, 256, 250), (3, 3, 7, 4), (2, 1, 512, 512)])
@pytest.mark.parametrize("T", [1, 37])
def test_geometries(T, hq, hkv, d, rotary, interleaved, dtype):
    _check(1, T, hq, hkv, d, rotary, dtype, interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pad,shift", [(64, 0), (5, 0), (3, 1), (6, 2), (4, 4), (0, 8)])
def test_strides_and_addresses(pad, shift, interleaved, dtype):
    _check(2, 19, 4, 2, 64, 64, dtype, interleaved, pad=pad, shift=shift, amplitude=1.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1023, 1024, 2050, 5000, 17000])
def test_many_tokens(T, dtype):
    _check(3, T, 2, 1, 64, 64, dtype, False)
    _check(4, T, 2, 1, 64, 32, dtype, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_positions(dtype):
    p = np.array([0, 1, 131071, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -1, -(1 << 31), -12345],
                 np.int32)
    _check(5, len(p), 3, 1, 128, 128, dtype, False, positions=p)
    _check(5, len(p), 3, 1, 128, 128, dtype, True, positions=p)


def test_the_widest_rows():
    _check(6, 3, 60, 4, 1024, 1024, "bf16", False)
    _check(6, 3, 1024, 1024, 32, 32, "fp16", True)


def test_position_zero_and_infinities():
    """Position 0 leaves the values; an infinity stays in its pair."""
    rng = np.random.default_rng(7)
    rows = _rows(rng, 2, 128, "f32")
    rows[1, 5] = np.inf
    freq, _ = kernels.rope_frequencies(64, 1e4)
    q, k = _launch(rows, np.array([0, 3], np.int32), freq, 1, 1, 64, 64, "f32")
    assert np.array_equal(q[0], rows[0, :64]) and np.array_equal(k[0], rows[0, 64:])
    bad = ~np.isfinite(q[1])
    assert bad[[5, 37]].all() and bad.sum() == 2 and np.isfinite(k[1]).all()


def test_a_captured_call_replays():
    rng = np.random.default_rng(8)
    T, hq, hkv, d = 50, 4, 2, 128
    stream = hip.Stream()
    rows = hip.DeviceBuffer.from_numpy(_rows(rng, T, (hq + hkv) * d, "bf16"))
    pos = hip.DeviceBuffer.from_numpy(rng.integers(0, 9999, T).astype(np.int32))
    freq = hip.DeviceBuffer.from_numpy(kernels.rope_frequencies(d, 1e6, "parts", 8.0, 4096)[0])
    out = hip.DeviceBuffer(T * (hq + hkv) * d * 2)

    def launch():
        w = (hq + hkv) * d
        kernels.launch_rope_packed(rows, rows.offset(hq * d * 2), out, out.offset(hq * d * 2), pos, freq,
                                   T, hq, hkv, d, d, False, 1.1, w, w, w, w, "bf16", stream)
        stream.synchronize()
        return out.to_numpy(np.uint16, (T, w))

    want = launch()
    graph = hip.Graph(stream)
    with graph:
        kernels.launch_rope_packed(rows, rows.offset(hq * d * 2), out, out.offset(hq * d * 2), pos, freq,
                                   T, hq, hkv, d, d, False, 1.1, 768, 768, 768, 768, "bf16", stream)
    for _ in range(3):
        out.fill(0xFF)
        hip.synchronize()
        graph.launch()
        stream.synchronize()
        assert np.array_equal(out.to_numpy(np.uint16, want.shape), want)
        assert np.array_equal(launch(), want)
