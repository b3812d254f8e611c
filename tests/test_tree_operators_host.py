"""Norms with rotary positions, e4m3 cache rows, attention of drafted tokens: what their entry points refuse
before they touch the device, and what is host arithmetic."""
import ctypes as C
import math

import numpy as np
import pytest

from logismos_amd import kernels
from tests import tree_reference as R

INVALID_VALUE = 1
P = C.c_void_p(4096)  # never read: the calls are refused


def _msg(check, *dims):
    msg = C.create_string_buffer(256)
    code = getattr(kernels.library(), check)(*dims, msg, len(msg))
    return code, msg.value.decode()


# ---------------------------------------------------------------------------- norms with rotary positions
NORM = dict(tokens=5, hq=4, hkv=2, d=64, rotary=64, axes=3, ps=5, qi=256, ki=128, qo=256, ko=128)


@pytest.mark.parametrize("change,frag", [
    (dict(tokens=0), "must be positive"), (dict(hq=0), "must be positive"), (dict(hkv=-1), "must not be negative"),
    (dict(tokens=(1 << 23) + 1, ps=(1 << 23) + 1), "exceeds"), (dict(d=0), "must be positive"),
    (dict(rotary=33), "rotary_dim"), (dict(rotary=66), "rotary_dim"), (dict(rotary=-2), "rotary_dim"),
    (dict(axes=0), "num_axes"), (dict(axes=256), "num_axes"), (dict(ps=4), "position_stride"),
    (dict(d=1026, rotary=64, qi=1 << 14, qo=1 << 14, ki=1 << 14, ko=1 << 14), "at most 1024"),
    (dict(qi=255), "q stride"), (dict(qo=255), "q stride"), (dict(ki=127), "k stride"), (dict(ko=127), "k stride"),
])
def test_norm_rope_shapes(change, frag):
    c = {**NORM, **change}
    code, msg = _msg("logismos_check_norm_rope_packed_shape", *c.values())
    assert code == INVALID_VALUE and frag in msg
    with pytest.raises(kernels.UnsupportedShape, match=frag):
        kernels.launch_norm_rope_packed(P, P, P, P, P, P, P, P, P, c["tokens"], c["hq"], c["hkv"], c["d"],
                                        c["rotary"], c["axes"], position_stride=c["ps"], q_in_stride=c["qi"],
                                        k_in_stride=c["ki"], q_out_stride=c["qo"], k_out_stride=c["ko"])


def test_norm_rope_shapes_that_are_fine():
    for change in (dict(), dict(axes=1, ps=0), dict(rotary=0, axes=0, ps=0), dict(hkv=0, ki=0, ko=0)):
        assert _msg("logismos_check_norm_rope_packed_shape", *{**NORM, **change}.values()) == (0, "")


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "f32"])
def test_norm_rope_arguments(dtype):
    far = [C.c_void_p(4096 + 65536 * i) for i in range(9)]
    names = ("q_in", "k_in", "q_out", "k_out", "positions", "axis_of_pair", "inv_freq", "q_gain", "k_gain")

    def refused(axes=3, **change):
        args = dict(zip(names, far))
        rest = {k: change.pop(k) for k in list(change) if k not in names}
        with pytest.raises(kernels.LaunchError, match="InvalidValue"):
            kernels.launch_norm_rope_packed(*{**args, **change}.values(), 5, 4, 2, 64, 64, axes, dtype=dtype, **rest)

    for name in ("q_in", "k_in", "q_out", "k_out", "positions", "axis_of_pair", "inv_freq"):
        refused(**{name: None})
    for name in ("q_in", "k_in", "q_out", "k_out"):
        refused(**{name: C.c_void_p(4097)})
    for name in ("positions", "q_gain", "k_gain", "inv_freq"):
        refused(**{name: C.c_void_p(4098)})
    for eps in (0.0, -1e-6, math.nan, math.inf):
        refused(eps=eps)
        refused(eps=eps, q_gain=None)
    for amplitude in (math.nan, math.inf):
        refused(amplitude=amplitude)
    refused(q_out=far[0], q_in_stride=320)  # one address with two strides
    refused(k_out=far[1], k_out_stride=320)
    with pytest.raises(ValueError):
        kernels.launch_norm_rope_packed(*far, 5, 4, 2, 64, 64, dtype="fp8")


# ---------------------------------------------------------------------------- e4m3 rows
ROWS = dict(tokens=5, hkv=2, d=64, block=16, blocks=4, ks=128, vs=128)


@pytest.mark.parametrize("change,frag", [
    (dict(tokens=-1), "total_tokens"), (dict(tokens=(1 << 23) + 1), "total_tokens"), (dict(hkv=0), "must be positive"),
    (dict(blocks=0), "must be positive"), (dict(d=48), "multiple of 32"), (dict(d=288, ks=576, vs=576), "multiple of 32"),
    (dict(block=24), "multiple of 16"), (dict(block=0), "multiple of 16"), (dict(block=1 << 16, blocks=1 << 16), "exceeds"),
    (dict(hkv=1 << 15, ks=1 << 21, vs=1 << 21), "exceeds"), (dict(ks=120), "smaller"), (dict(vs=64), "smaller"),
    (dict(ks=132), "multiples of 8"), (dict(vs=129), "multiples of 8"),
])
def test_kv_e4m3_shapes(change, frag):
    c = {**ROWS, **change}
    code, msg = _msg("logismos_check_kv_e4m3_shape", *c.values())
    assert code == INVALID_VALUE and frag in msg
    for call in (kernels.launch_kv_write_e4m3, kernels.launch_kv_gather_e4m3):
        with pytest.raises(kernels.UnsupportedShape, match=frag):
            call(P, P, P, P, P, P, P, *c.values())


def test_kv_e4m3_arguments():
    calls = [lambda *a, b=b: kernels.launch_kv_write_e4m3(*a, 5, 2, 64, 16, 4, bf16=b) for b in (False, True)]
    calls += [lambda *a, t=t: kernels.launch_kv_gather_e4m3(*a, 5, 2, 64, 16, 4, dtype=t)
              for t in ("fp16", "bf16", "f32")]
    for call in calls:
        for at in range(7):
            for bad in (None, C.c_void_p(4100)):  # (slots: 8 bytes)
                with pytest.raises(kernels.LaunchError, match="InvalidValue"):
                    call(*[bad if i == at else P for i in range(7)])
    with pytest.raises(ValueError):
        kernels.launch_kv_gather_e4m3(P, P, P, P, P, P, P, 5, 2, 64, 16, 4, dtype="int8")


def test_no_rows_are_fine_without_a_device():
    kernels.launch_kv_write_e4m3(None, None, None, None, None, None, None, 0, 2, 64, 16, 4)
    kernels.launch_kv_gather_e4m3(None, None, None, None, None, None, None, 0, 2, 64, 16, 4)


def test_the_reference_rounds_as_the_type_does():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(0)
    values = R.e4m3_values(np.arange(127).astype(np.uint8))
    x = np.concatenate([values, (values[1:] + values[:-1]) / 2, rng.uniform(-448, 448, 4000),
                        rng.standard_normal(4000) * 2.0 ** rng.integers(-12, 8, 4000)])
    x = np.concatenate([x, -x]).clip(-448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn)
    assert np.array_equal(R.e4m3_codes(x.astype(np.float64)), want.view(torch.uint8).numpy())
    codes = np.arange(256).astype(np.uint8)
    assert np.array_equal(R.e4m3_values(codes), torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy(),
                          equal_nan=True)


def test_exponents_of_rows():
    rows = np.array([[448.0, 1], [449.0, 1], [1.75, 0], [1.7501, 0], [0, 0], [2.0 ** -120, 0], [1e30, -5],
                     [np.inf, 3.5], [np.nan, -896]])
    codes, e = R.quantise(rows)
    assert e.tolist() == [0, 1, -8, -7, -64, -64, 32, -7, 1]
    assert codes[0].tolist() == [0x7E, 0x38] and codes[7, 0] == 0x7F and codes[6, 0] == 0x7E and codes[8, 1] == 0xFE


# ---------------------------------------------------------------------------- tree attention
TREE = dict(num_seqs=2, total=10, max_q=6, hq=8, hkv=2, d=64, block=16, per_seq=8, blocks=20, words=1, qs=512, os=512)


@pytest.mark.parametrize("change,frag", [
    (dict(num_seqs=0), "must be positive"), (dict(total=0), "must be positive"), (dict(max_q=0), "must be positive"),
    (dict(num_seqs=65536), "<= 65535"), (dict(total=65536), "<= 65535"), (dict(max_q=11), "exceeds total_tokens"),
    (dict(hq=0), "must be positive"), (dict(hkv=0), "must be positive"), (dict(hq=7), "not a multiple"),
    (dict(d=80), "multiple of 32"), (dict(d=288), "multiple of 32"), (dict(block=24), "multiple of 16"),
    (dict(per_seq=0), "must be positive"), (dict(blocks=0), "must be positive"),
    (dict(per_seq=1 << 27), "exceeds"), (dict(blocks=1 << 27), "exceeds"),
    (dict(words=0), "mask_words"), (dict(words=5), "mask_words"), (dict(total=100, max_q=65), "mask_words"),
    (dict(hq=1 << 15, hkv=1 << 15, qs=1 << 21, os=1 << 21), "exceeds"),
    (dict(qs=504), "smaller"), (dict(os=504), "smaller"), (dict(qs=516), "multiples of 8"),
    (dict(os=514), "multiples of 8"), (dict(os=(1 << 22) + 8), "at most"),
    (dict(num_seqs=60000, total=60000, max_q=1, per_seq=1 << 20), "too many key tiles"),
])
def test_tree_shapes(change, frag):
    c = {**TREE, **change}
    code, msg = _msg("logismos_check_paged_attn_tree_shape", *c.values())
    assert code == INVALID_VALUE and frag in msg
    for exp, bf16 in ((None, False), (P, False), (P, True)):
        with pytest.raises(kernels.UnsupportedShape, match=frag):
            kernels.launch_paged_attn_tree(P, P, P, P, P, P, P, P, P, c["num_seqs"], c["total"], c["max_q"], c["hq"],
                                           c["hkv"], c["d"], c["block"], c["per_seq"], c["blocks"], 0.125, c["words"],
                                           exp, exp, c["qs"], c["os"], bf16)


def test_tree_arguments():
    names = ("q", "k_pool", "v_pool", "block_tables", "cu", "ctx", "mask", "out", "workspace")
    for exps in ((None, None), (P, P)):
        def refused(scale=0.125, exps=exps, **change):
            with pytest.raises(kernels.LaunchError, match="InvalidValue"):
                kernels.launch_paged_attn_tree(*{**dict.fromkeys(names, P), **change}.values(), 2, 10, 6, 8, 2, 64, 16,
                                               8, 20, scale, k_exp=exps[0], v_exp=exps[1])

        for name in names:
            refused(**{name: None})
            refused(**{name: C.c_void_p(4098)})
        refused(mask=C.c_void_p(4100))
        for name in ("q", "k_pool", "v_pool", "out", "workspace"):
            refused(**{name: C.c_void_p(4104)})
        for scale in (0.0, -1.0, math.inf, math.nan, 3e38):
            refused(scale=scale)
        refused(exps=(P, None))
        refused(exps=(None, P))
        refused(exps=(C.c_void_p(4104), P))
    with pytest.raises(ValueError):
        kernels.launch_paged_attn_tree(*[P] * 9, 2, 10, 6, 8, 2, 64, 16, 8, 20, 0.125, bf16=True)


def test_tree_workspace():
    ws = kernels.paged_attn_tree_workspace_bytes
    assert ws(10, 6, 8, 2, 64) % 16 == 0 and 0 < ws(10, 6, 8, 2, 64) <= ws(100, 60, 8, 2, 64)
    # (a bound that does not depend on how many tokens there are beyond the longest tree)
    assert ws(100, 60, 8, 2, 64) == ws(1000, 60, 8, 2, 64)
    for bad in ((0, 1, 8, 2, 64), (4, 5, 8, 2, 64), (4, 4, 7, 2, 64), (4, 4, 8, 0, 64), (4, 4, 8, 2, 0)):
        assert ws(*bad) == 0


@pytest.mark.parametrize("n,words", [(1, 1), (2, 1), (64, 1), (65, 2), (200, 4), (256, 4), (7, 3)])
def test_tree_mask(n, words):
    rng = np.random.default_rng(n)
    parents = np.array([-1 if i == 0 or rng.random() < 0.1 else rng.integers(0, i) for i in range(n)])
    got = kernels.tree_mask(parents, words)
    assert np.array_equal(got, R.mask_bits(R.ancestors(parents), words))
    assert np.array_equal(kernels.tree_mask(parents), R.mask_bits(R.ancestors(parents), (n + 63) // 64))
    chain = kernels.tree_mask(np.arange(n) - 1, words)
    assert np.array_equal(chain, R.mask_bits(np.tri(n, dtype=bool), words))


def test_the_mask_of_no_tokens():
    assert kernels.tree_mask([]).shape == (0, 1) and kernels.tree_mask([], 3).shape == (0, 3)


@pytest.mark.parametrize("parents,words", [([0], 1), ([-2], 1), ([-1, 1], 1), ([-1, 2, 0], 1), ([], 5),
                                           ([-1] * 65, 1), ([-1] * 257, 0), ([-1], 5), ([-1], -1)])
def test_trees_that_are_none(parents, words):
    with pytest.raises(kernels.UnsupportedShape):
        kernels.tree_mask(parents, words)
