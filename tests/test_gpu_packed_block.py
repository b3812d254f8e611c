"""The attention half of a block over packed rows, as a program calls it: the shared projection over
4-bit weights, each request's adapter on top of it, rotary positions in place, attention of the packed
sequences over columns of the same rows.  Every stage against the 64-bit form of what it was given, and
the whole run captured and replayed against the stages."""
import numpy as np
import pytest

import oracle as O
from logismos_amd import hip, kernels
from tests import packed_reference as R

pytestmark = pytest.mark.gpu


def _up(a):
    return hip.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


@pytest.mark.parametrize("hidden,hq,hkv,d,rotary,interleaved,causal", [
    (896, 14, 2, 64, 64, False, True), (1536, 12, 2, 128, 64, True, False),
    (512, 8, 8, 64, 32, False, True)])
def test_block(hidden, hq, hkv, d, rotary, interleaved, causal):
    rng = np.random.default_rng(1)
    lens, pick, ranks = [70, 1, 33, 129], [1, 0, -1, 2], [8, 24, 5]
    T, width, r = sum(lens), (hq + 2 * hkv) * d, 24
    x = R.to_bits(rng.standard_normal((T, hidden), np.float32), "bf16")
    w = rng.standard_normal((width, hidden), np.float32) * np.float32(hidden ** -0.5)
    qw, scale, zero = O.quantize_q4g128(w, width, hidden)
    a = R.to_bits(rng.standard_normal((3, r, hidden), np.float32) * np.float32(hidden ** -0.5), "bf16")
    b = R.to_bits(rng.standard_normal((3, width, r), np.float32) * np.float32(0.2), "bf16")
    gain = np.array([0.5, 1.0, 2.0], np.float32)
    positions = np.concatenate([np.arange(n) + 1000 * i for i, n in enumerate(lens)]).astype(np.int32)
    freq, amplitude = kernels.rope_frequencies(rotary, 1e6, "parts", 4.0, 512)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    stream = hip.Stream()
    d_x, d_qw, d_sc, d_ze = _up(x), _up(qw), _up(scale), _up(zero)
    d_a, d_b, d_ranks, d_gain = _up(a), _up(b), _up(np.array(ranks, np.int32)), _up(gain)
    d_pick, d_cu, d_pos, d_f = _up(np.array(pick, np.int32)), _up(cu), _up(positions), _up(freq)
    rows, out = hip.DeviceBuffer(T * width * 2), hip.DeviceBuffer(T * hq * d * 2)
    ws = hip.DeviceBuffer(kernels.adapter_add_workspace_bytes(T, r))
    k_at, v_at = rows.offset(2 * hq * d), rows.offset(2 * (hq + hkv) * d)

    def project():
        kernels.launch_qgemm_q4g128_bf16(d_x, d_qw, d_sc, d_ze, rows, T, width, hidden, stream)

    def adapt():
        kernels.launch_adapter_add(d_x, d_a, d_b, d_ranks, d_gain, d_pick, d_cu, rows, rows, ws, 4, T, 3, r,
                                   width, hidden, bf16=True, stream=stream)

    def rotate():
        kernels.launch_rope_packed(rows, k_at, rows, k_at, d_pos, d_f, T, hq, hkv, d, rotary, interleaved,
                                   amplitude, width, width, width, width, "bf16", stream)

    def attend():
        kernels.launch_attn_packed(rows, k_at, v_at, d_cu, out, 4, T, hq, hkv, d, d ** -0.5, causal, width,
                                   width, width, bf16=True, stream=stream)

    def read(buf, n):
        stream.synchronize()
        return buf.to_numpy(np.uint16, (T, n))

    f = lambda v: R.from_bits(v, "bf16")  # noqa: E731
    project()
    base = read(rows, width).copy()
    adapt()
    adapted = read(rows, width).copy()
    R.assert_within(f(adapted), *R.adapter(f(x), f(a), f(b), ranks, gain, pick, lens, f(base), "bf16", "bf16"),
                    what="adapters")
    rotate()
    turned = read(rows, width).copy()
    qk = f(adapted[:, :(hq + hkv) * d]).reshape(T, hq + hkv, d)
    want, bound = R.rope(qk, positions, freq, rotary, interleaved, amplitude, "bf16")
    R.assert_within(f(turned[:, :(hq + hkv) * d]), want.reshape(T, -1), bound.reshape(T, -1), what="rope")
    assert np.array_equal(turned[:, (hq + hkv) * d:], adapted[:, (hq + hkv) * d:])
    attend()
    got = read(out, hq * d).copy()
    q, k, v = np.split(f(turned).reshape(T, -1, d), [hq, hq + hkv], 1)
    want, bound = R.attention(q, k, v, lens, d ** -0.5, causal, "bf16")
    R.assert_within(f(got), want.reshape(T, -1), bound.reshape(T, -1), what="attention")

    graph = hip.Graph(stream)
    with graph:
        project()
        adapt()
        rotate()
        attend()
    for _ in range(3):
        out.fill(0xFF)
        hip.synchronize()
        graph.launch()
        assert np.array_equal(read(out, hq * d), got)
        assert np.array_equal(read(rows, width), turned)
        project()
        stream.synchronize()
