"""Operators over packed rows where rows lie so far apart that offsets pass 32 bits, and two calls of one
operator at the same time."""
import ctypes as C

import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as R

pytestmark = pytest.mark.gpu

STRIDE = 1 << 20  # elements of 16 bits: 2100 rows are 4.4 GB
ROWS = 2100


class Far:
    """ROWS rows of STRIDE elements; columns of it as arrays."""

    def __init__(self):
        free, _ = hip.mem_info()
        if free < (6 << 30):
            pytest.skip("less than 6 GiB free")
        self.buf = hip.DeviceBuffer(ROWS * STRIDE * 2)

    def _copy(self, host, column, to_device):
        width, rows = host.shape[1] * host.dtype.itemsize, host.shape[0]
        dev, h = self.buf.offset(2 * column), host.ctypes.data_as(C.c_void_p)
        args = (dev, C.c_size_t(2 * STRIDE), h, C.c_size_t(width)) if to_device else \
            (h, C.c_size_t(width), dev, C.c_size_t(2 * STRIDE))
        hip.check(hip._runtime().hipMemcpy2D(*args, C.c_size_t(width), C.c_size_t(rows),
                                             C.c_int(1 if to_device else 2)), "hipMemcpy2D")

    def put(self, column, host):
        self._copy(np.ascontiguousarray(host), column, True)
        return self.buf.offset(2 * column)

    def get(self, column, width, dtype=np.uint16):
        out = np.empty((ROWS, width), dtype)
        hip.synchronize()
        self._copy(out, column, False)
        return out


def test_rows_far_apart():
    rng = np.random.default_rng(1)
    far = Far()
    f = lambda v: R.from_bits(v, "bf16")  # noqa: E731
    hq, hkv, d, k, r = 4, 2, 64, 256, 16
    lens, pick, ranks = [ROWS - 700, 699, 1], [1, -1, 0], [16, 9]
    width = (hq + 2 * hkv) * d
    x = R.to_bits(rng.standard_normal((ROWS, k), np.float32), "bf16")
    rows = R.to_bits(rng.standard_normal((ROWS, width), np.float32), "bf16")
    a = R.to_bits(rng.standard_normal((2, r, k), np.float32) / 16, "bf16")
    b = R.to_bits(rng.standard_normal((2, width, r), np.float32) / 4, "bf16")
    d_x, d_rows = far.put(0, x), far.put(1024, rows)
    up = hip.DeviceBuffer.from_numpy
    cu = up(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    ws = hip.DeviceBuffer(kernels.adapter_add_workspace_bytes(ROWS, r))
    keep = [up(a), up(b), up(np.array(ranks, np.int32)), up(np.array([1.0, 2.0], np.float32)),
            up(np.array(pick, np.int32))]
    kernels.launch_adapter_add(d_x, *keep, cu, d_rows, d_rows, ws, 3, ROWS, 2, r, width, k, STRIDE, STRIDE,
                               STRIDE, bf16=True)
    got = far.get(1024, width)
    R.assert_within(f(got), *R.adapter(f(x), f(a), f(b), ranks, [1.0, 2.0], pick, lens, f(rows), "bf16", "bf16"))
    rows = got

    positions = rng.integers(0, 5000, ROWS).astype(np.int32)
    freq, _ = kernels.rope_frequencies(d, 1e4)
    at = [far.buf.offset(2 * (1024 + c * d)) for c in (0, hq, hq + hkv)]
    kernels.launch_rope_packed(at[0], at[1], at[0], at[1], up(positions), up(freq), ROWS, hq, hkv, d, d, False, 1.0,
                               STRIDE, STRIDE, STRIDE, STRIDE, "bf16")
    got = far.get(1024, width)
    qk = f(rows[:, :(hq + hkv) * d]).reshape(ROWS, -1, d)
    want, bound = R.rope(qk, positions, freq, d, False, 1.0, "bf16")
    R.assert_within(f(got[:, :(hq + hkv) * d]), want.reshape(ROWS, -1), bound.reshape(ROWS, -1))
    assert np.array_equal(got[:, (hq + hkv) * d:], rows[:, (hq + hkv) * d:])
    rows = got

    out_at = 4096
    kernels.launch_attn_packed(*at, cu, far.buf.offset(2 * out_at), 3, ROWS, hq, hkv, d, 0.125, True, STRIDE,
                               STRIDE, STRIDE, STRIDE, bf16=True)
    got = far.get(out_at, hq * d)
    q, kk, v = np.split(f(rows).reshape(ROWS, -1, d), [hq, hq + hkv], 1)
    want, bound = R.attention(q, kk, v, lens, 0.125, True, "bf16")
    R.assert_within(f(got), want.reshape(ROWS, -1), bound.reshape(ROWS, -1))


def test_adapters_on_two_streams_at_once():
    rng = np.random.default_rng(2)
    up = hip.DeviceBuffer.from_numpy
    runs = []
    for n, k, T in ((520, 384, 700), (2048, 512, 40)):
        x, base = (R.to_bits(rng.standard_normal((T, w), np.float32), "fp16") for w in (k, n))
        a = R.to_bits(rng.standard_normal((2, 32, k), np.float32) / 20, "fp16")
        b = R.to_bits(rng.standard_normal((2, n, 32), np.float32) / 5, "fp16")
        lens, pick = [T - 5, 5], [1, 0]
        want = R.adapter(*(R.from_bits(v, "fp16") for v in (x, a, b)), [32, 20], [0.5, 1.5], pick, lens,
                         R.from_bits(base, "fp16"), "fp16", "fp16")
        bufs = [up(v) for v in (x, a, b, np.array([32, 20], np.int32), np.array([0.5, 1.5], np.float32),
                                np.array(pick, np.int32), np.array([0, T - 5, T], np.int32), base)]
        runs.append((bufs, hip.DeviceBuffer(T * n * 2),
                     hip.DeviceBuffer(kernels.adapter_add_workspace_bytes(T, 32)), hip.Stream(), n, k, T, want))
    for _ in range(5):
        for bufs, out, ws, stream, n, k, T, _w in runs:
            kernels.launch_adapter_add(*bufs, out, ws, 2, T, 2, 32, n, k, stream=stream)
    for _b, out, _ws, stream, n, _k, T, want in runs:
        stream.synchronize()
        R.assert_within(R.from_bits(out.to_numpy(np.float16, (T, n)), "fp16"), *want)


def test_rope_on_two_streams_at_once():
    rng = np.random.default_rng(3)
    up = hip.DeviceBuffer.from_numpy
    freq, _ = kernels.rope_frequencies(64, 1e4)
    d_f = up(freq)
    runs = []
    for T in (3000, 17):
        x = R.to_bits(rng.standard_normal((T, 3 * 64), np.float32), "fp16")
        p = rng.integers(0, 9000, T).astype(np.int32)
        want = R.rope(R.from_bits(x, "fp16").reshape(T, 3, 64), p, freq, 64, True, 1.0, "fp16")
        runs.append((up(x), up(p), hip.DeviceBuffer(T * 384), hip.Stream(), T, want))
    for _ in range(5):
        for x, p, out, stream, T, _w in runs:
            kernels.launch_rope_packed(x, None, out, None, p, d_f, T, 3, 0, 64, 64, True, stream=stream)
    for _x, _p, out, stream, T, want in runs:
        stream.synchronize()
        R.assert_within(R.from_bits(out.to_numpy(np.float16, (T, 3, 64)), "fp16"), *want)
