"""RMS norms of heads at the ends of the ranges: rows and gains whose quotient is no ordinary number of 32 bits."""
import numpy as np
import pytest

from logismos_amd import kernels
from tests import packed_reference as P
from tests.test_gpu_norm_rope_packed import _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rotary", [0, 64])
@pytest.mark.parametrize("d", [64, 1000])
@pytest.mark.parametrize("size", [2.0 ** 80, 2.0 ** 100, 2.0 ** 122])
@pytest.mark.parametrize("gain", [2.0 ** -30, 2.0 ** -12, 1.0, 2.0 ** 40])
def test_large_rows_with_small_and_large_gains(gain, size, d, rotary, dtype):
    """The quotient of gain and root is far below the smallest ordinary number of fp32 where the result is not."""
    rng = np.random.default_rng(d)
    T, hq, hkv = 3, 2, 1
    rows = P.to_bits(rng.uniform(-1, 1, (T, 3 * d)) * size, dtype)
    gains = [(rng.uniform(0.5, 2, d) * gain).astype(np.float32) for _ in range(2)]
    positions = rng.integers(0, 1000, (1, T)).astype(np.int32)
    freq = kernels.rope_frequencies(rotary, 1e4)[0] if rotary else None
    axis = np.zeros(rotary // 2, np.uint8)
    x = P.from_bits(rows, dtype).reshape(T, 3, d)
    want, bound = _want(x, gains, positions, axis, freq, hq, rotary, False, 1.0, dtype)
    out = _run(rows, positions, None, freq, gains, hq, hkv, d, rotary, dtype)
    for o, at in zip(out, (slice(0, hq * d), slice(hq * d, 3 * d))):
        P.assert_within(P.from_bits(o[:T], dtype), want[:, at], bound[:, at])
