"""Operators over packed rows: what their entry points refuse before they touch the device, and the
frequencies of rotary positions, which are host arithmetic."""
import ctypes as C
import math

import numpy as np
import pytest

from logismos_amd import kernels

INVALID_VALUE = 1
P = C.c_void_p(4096)  # never read: the calls are refused


def _msg(check, *dims):
    msg = C.create_string_buffer(256)
    code = getattr(kernels.library(), check)(*dims, msg, len(msg))
    return code, msg.value.decode()


# ---------------------------------------------------------------------------- attention
ATTN = dict(num_seqs=2, total=10, hq=8, hkv=2, d=64, qs=512, ks=128, vs=128, os=512)


@pytest.mark.parametrize("change,frag", [
    (dict(num_seqs=0), "must be positive"), (dict(total=0), "must be positive"),
    (dict(hq=0), "must be positive"), (dict(hkv=-1), "must be positive"),
    (dict(hq=7), "not a multiple of num_kv_heads"), (dict(d=80), "multiple of 32 up to 256"),
    (dict(d=288, qs=8 * 288, os=8 * 288, ks=576, vs=576), "multiple of 32 up to 256"),
    (dict(total=1 << 24), "exceeds"), (dict(total=1 << 23, num_seqs=(1 << 23) + 1), "exceeds"),
    (dict(total=1 << 22, hq=256, hkv=2, qs=16384, os=16384), "exceeds"),
    (dict(total=1 << 22, num_seqs=1 << 22, hkv=8, ks=512, vs=512), "exceeds"),
    (dict(qs=504), "smaller than its row"), (dict(os=504), "smaller than its row"),
    (dict(ks=120), "smaller than its row"), (dict(vs=120), "smaller than its row"),
    (dict(qs=516), "multiples of 8"), (dict(vs=130), "multiples of 8"),
    (dict(ks=(1 << 22) + 8), "at most"), (dict(os=(1 << 22) + 8), "at most"),
])
def test_attn_packed_shapes(change, frag):
    code, msg = _msg("logismos_check_attn_packed_shape", *{**ATTN, **change}.values())
    assert code == INVALID_VALUE and frag in msg
    c = {**ATTN, **change}
    with pytest.raises(kernels.UnsupportedShape, match=frag):
        kernels.launch_attn_packed(P, P, P, P, P, c["num_seqs"], c["total"], c["hq"], c["hkv"],
                                   c["d"], 0.125, True, c["qs"], c["ks"], c["vs"], c["os"])


@pytest.mark.parametrize("bf16", [False, True])
def test_attn_packed_arguments(bf16):
    def refused(q=P, k=P, v=P, cu=P, out=P, scale=0.125):
        with pytest.raises(kernels.LaunchError, match="InvalidValue"):
            kernels.launch_attn_packed(q, k, v, cu, out, 2, 10, 8, 2, 64, scale, bf16=bf16)

    for name in ("q", "k", "v", "out"):
        refused(**{name: None})
        refused(**{name: C.c_void_p(4104)})
    refused(cu=None)
    refused(cu=C.c_void_p(4098))
    for scale in (0.0, -1.0, math.inf, math.nan, 3e38):
        refused(scale=scale)


# ---------------------------------------------------------------------------- rotary positions
ROPE = dict(tokens=5, hq=4, hkv=2, d=64, rotary=64, qi=256, ki=128, qo=256, ko=128)


@pytest.mark.parametrize("change,frag", [
    (dict(tokens=0), "must be positive"), (dict(hq=0), "must be positive"),
    (dict(tokens=(1 << 23) + 1), "exceeds"), (dict(d=0), "must be positive"), (dict(hkv=-1), "must not be negative"),
    (dict(rotary=0), "rotary_dim"), (dict(rotary=33), "rotary_dim"), (dict(rotary=66), "rotary_dim"),
    (dict(d=1026, rotary=64, qi=1 << 14, qo=1 << 14, ki=1 << 14, ko=1 << 14), "at most 1024"),
    (dict(hq=1024, hkv=1, qi=65536, qo=65536), "exceeds 65536"),
    (dict(qi=255), "q stride"), (dict(qo=255), "q stride"), (dict(ki=127), "k stride"),
    (dict(ko=127), "k stride"),
])
def test_rope_packed_shapes(change, frag):
    code, msg = _msg("logismos_check_rope_packed_shape", *{**ROPE, **change}.values())
    assert code == INVALID_VALUE and frag in msg


def test_rope_packed_without_k_looks_at_no_k_stride():
    assert _msg("logismos_check_rope_packed_shape",
                *{**ROPE, "hkv": 0, "ki": -1, "ko": 0}.values())[0] == 0


@pytest.mark.parametrize("dtype,size", [("fp16", 2), ("bf16", 2), ("f32", 4)])
def test_rope_packed_arguments(dtype, size):
    def refused(qi=P, ki=P, qo=P, ko=P, pos=P, freq=P, amplitude=1.0):
        with pytest.raises(kernels.LaunchError, match="InvalidValue"):
            kernels.launch_rope_packed(qi, ki, qo, ko, pos, freq, 5, 4, 2, 64, 64,
                                       amplitude=amplitude, dtype=dtype)

    for name in ("qi", "ki", "qo", "ko"):
        refused(**{name: None})
        refused(**{name: C.c_void_p(4096 + size // 2)})
    refused(pos=None)
    refused(pos=C.c_void_p(4098))
    refused(freq=None)
    refused(freq=C.c_void_p(4100))
    refused(amplitude=math.inf)
    refused(amplitude=math.nan)
    with pytest.raises(ValueError):
        kernels.launch_rope_packed(P, P, P, P, P, P, 5, 4, 2, 64, 64, dtype="f64")


@pytest.mark.parametrize("rotary", [2, 6, 64, 128])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("base", 8.0),
                                            ("parts", 16.0), ("parts", 1.0)])
def test_rope_frequencies(rotary, scaling, factor):
    if scaling == "base" and rotary == 2:
        with pytest.raises(kernels.UnsupportedShape):
            kernels.rope_frequencies(rotary, 1e4, scaling, factor)
        return
    f, amplitude = kernels.rope_frequencies(rotary, 1e4, scaling, factor, 4096)
    i = np.arange(rotary // 2)
    plain = np.exp(-2 * i / rotary * np.log(1e4))
    if scaling == "linear":
        want = plain / factor
    elif scaling == "base":
        want = np.exp(-2 * i / rotary * (np.log(1e4) + rotary / (rotary - 2) * np.log(factor)))
    elif scaling == "parts":
        turns = 4096 * plain / (2 * np.pi)
        keep = np.clip((turns - 1) / 31, 0, 1)
        want = plain * keep + plain / factor * (1 - keep)
    else:
        want = plain
    assert np.allclose(f, want, rtol=1e-13, atol=0)  # (some ten roundings of 2^-53, times the logarithm)
    assert amplitude == np.float32(0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0)
    if scaling == "base":  # the ends the changed base is made for
        assert np.isclose(f[-1], plain[-1] / factor, rtol=1e-12) and f[0] == 1.0


@pytest.mark.parametrize("args", [
    dict(rotary=0), dict(rotary=-2), dict(rotary=7), dict(rotary=1026), dict(base=0.0), dict(base=-1.0),
    dict(base=math.nan), dict(base=math.inf), dict(scaling="linear", factor=0.5),
    dict(scaling="linear", factor=math.nan), dict(scaling="base", factor=math.inf),
    dict(scaling="parts", original=0), dict(scaling="parts", fast=1.0),
    dict(scaling="parts", slow=-1.0), dict(scaling="parts", fast=math.inf),
])
def test_rope_frequencies_refusals(args):
    a = {**dict(rotary=64, base=1e4, scaling="none", factor=2.0, original=4096, fast=32.0, slow=1.0),
         **args}
    with pytest.raises(kernels.UnsupportedShape):
        kernels.rope_frequencies(a["rotary"], a["base"], a["scaling"], a["factor"], a["original"],
                                 a["fast"], a["slow"])


def test_rope_frequencies_unknown_scaling():
    with pytest.raises(ValueError):
        kernels.rope_frequencies(64, 1e4, "cubic")
    out, amp = (C.c_double * 32)(), C.c_float()
    for scaling in (-1, 4):
        assert kernels.library().logismos_rope_frequencies(
            C.cast(out, C.c_void_p), C.byref(amp), 64, 1e4, scaling, 2.0, 4096, 32.0, 1.0) == 1
    assert kernels.library().logismos_rope_frequencies(None, C.byref(amp), 64, 1e4, 0, 2.0, 4096,
                                                       32.0, 1.0) == 1


# ---------------------------------------------------------------------------- adapters
ADAPTER = dict(num_seqs=2, total=10, adapters=3, max_rank=16, n=64, k=128, xs=128, bs=64, os=64)


@pytest.mark.parametrize("change,frag", [
    (dict(num_seqs=0), "must be positive"), (dict(total=0), "must be positive"),
    (dict(adapters=0), "must be positive"), (dict(n=0), "must be positive"),
    (dict(k=-8), "must be positive"), (dict(max_rank=0), "max_rank"), (dict(max_rank=12), "max_rank"),
    (dict(max_rank=264), "max_rank"), (dict(n=60), "multiples of 8"), (dict(k=124), "multiples of 8"),
    (dict(xs=120), "smaller than its row"), (dict(bs=56), "smaller than its row"),
    (dict(os=56), "smaller than its row"), (dict(xs=132), "strides must be multiples of 8"),
    (dict(os=68), "strides must be multiples of 8"), (dict(total=1 << 24), "exceeds"),
    (dict(n=1 << 23, bs=1 << 23, os=1 << 23), "n and k must be at most"),
    (dict(k=1 << 23, xs=1 << 23), "n and k must be at most"),
    (dict(bs=(1 << 22) + 8), "base and out strides"), (dict(os=(1 << 22) + 8), "base and out strides"),
])
def test_adapter_add_shapes(change, frag):
    code, msg = _msg("logismos_check_adapter_add_shape", *{**ADAPTER, **change}.values())
    assert code == INVALID_VALUE and frag in msg


@pytest.mark.parametrize("bf16", [False, True])
def test_adapter_add_arguments(bf16):
    names = ("x", "a", "b", "ranks", "scales", "adapter_of_seq", "cu", "base", "out", "ws")

    def refused(os=64, **other):
        args = [other.get(n, C.c_void_p(4096 + 65536 * i)) for i, n in enumerate(names)]
        with pytest.raises(kernels.LaunchError, match="InvalidValue"):
            kernels.launch_adapter_add(*args, 2, 10, 3, 16, 64, 128, out_stride=os, bf16=bf16)

    for name in names:
        refused(**{name: None})
        refused(**{name: C.c_void_p(4098)})
    for name in ("x", "a", "b", "base", "out", "ws"):
        refused(**{name: C.c_void_p(4104)})
    refused(base=P, out=P, os=72)  # one address with two strides is not in place


def test_adapter_add_workspace():
    size = kernels.adapter_add_workspace_bytes
    assert size(0, 8) == 0 and size(8, 0) == 0 and size(-1, 8) == 0
    assert size(1, 8) >= 32 and size(1 << 23, 256) > 1 << 32
