"""Rotary positions of packed rows: calls that are refused, beside those for shapes, addresses and types."""
import ctypes as C

import pytest

from logismos_amd import kernels

Q, K, POS, F = (C.c_void_p(4096 + 65536 * i) for i in range(4))  # never read: the calls are refused


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "f32"])
@pytest.mark.parametrize("strides", [dict(q_in_stride=320), dict(q_out_stride=320), dict(k_in_stride=192),
                                     dict(k_out_stride=192), dict(q_in_stride=264, q_out_stride=256)])
def test_one_address_with_two_strides_is_not_in_place(strides, dtype):
    with pytest.raises(kernels.LaunchError, match="InvalidValue"):
        kernels.launch_rope_packed(Q, K, Q, K, POS, F, 5, 4, 2, 64, 64, dtype=dtype, **strides)


@pytest.mark.parametrize("rotary,base,scaling,factor", [
    (128, 5e-324, "none", 1.0), (128, 5e-324, "linear", 4.0), (128, 5e-324, "parts", 4.0),  # frequencies beyond 64 bits
    (4, 1e4, "base", 1e200), (64, 1e300, "base", 1e30)])  # a base that is
def test_frequencies_that_are_not_finite(rotary, base, scaling, factor):
    with pytest.raises(kernels.UnsupportedShape):
        kernels.rope_frequencies(rotary, base, scaling, factor, 4096)


def test_frequencies_of_a_base_below_one():
    f, _ = kernels.rope_frequencies(8, 1e-4)
    assert abs(f - [1.0, 10.0, 100.0, 1000.0]).max() < 1e-10
