"""Cache rows in e4m3: what is written and what is read back, bit for bit against the 64-bit form."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as P
from tests import tree_reference as R

pytestmark = pytest.mark.gpu


class Pools:
    """Pools full of a pattern, so that a byte which should not have been written is seen."""

    def __init__(self, blocks, block, hkv, d, fill=0x5A):
        self.shape, self.exps = (blocks, block, hkv, d), (blocks, hkv, block)
        self.k, self.v = (hip.DeviceBuffer(blocks * block * hkv * d) for _ in range(2))
        self.k_exp, self.v_exp = (hip.DeviceBuffer(blocks * block * hkv) for _ in range(2))
        for b in (self.k, self.v, self.k_exp, self.v_exp):
            b.fill(fill)

    def rows(self):
        """[(codes [rows][hkv][d], exponent bytes [rows][hkv])] of K and V."""
        hip.synchronize()
        n = self.shape[0] * self.shape[1]
        return [(p.to_numpy(np.uint8, self.shape).reshape(n, *self.shape[2:]),
                 e.to_numpy(np.uint8, self.exps).transpose(0, 2, 1).reshape(n, -1))
                for p, e in ((self.k, self.k_exp), (self.v, self.v_exp))]


def _slots(rng, tokens, rows):
    """Distinct slots, a few of them none."""
    s = rng.permutation(rows)[:tokens].astype(np.int64)
    s[rng.random(tokens) < 0.1] = rng.choice([-1, rows, 1 << 40, -(1 << 40)])
    return s


def _write(x, hkv, d, slots, pools, dtype, offset=0, stream=None):
    """x: bits of rows that hold K at `offset` and V behind it."""
    rows, at = hip.DeviceBuffer.from_numpy(x), hip.DeviceBuffer.from_numpy(slots)
    width, block, blocks = x.shape[1], pools.shape[1], pools.shape[0]
    kernels.launch_kv_write_e4m3(rows.offset(2 * offset), rows.offset(2 * (offset + hkv * d)), pools.k, pools.k_exp,
                                 pools.v, pools.v_exp, at, len(slots), hkv, d, block, blocks, width, width,
                                 dtype == "bf16", stream)
    hip.synchronize()


def _check_write(x, hkv, d, slots, pools, dtype, offset=0, fill=0x5A):
    _write(x, hkv, d, slots, pools, dtype, offset)
    n = pools.shape[0] * pools.shape[1]
    real = (slots >= 0) & (slots < n)
    for which, (codes, exps) in enumerate(pools.rows()):
        a = offset + which * hkv * d
        want, e = R.quantise(P.from_bits(x[:, a:a + hkv * d], dtype).reshape(-1, hkv, d))
        other = np.ones(n, bool)
        other[slots[real]] = False
        assert np.array_equal(exps[slots[real]], (e[real] + 127).astype(np.uint8))
        nan = (want & 0x7F) == 0x7F  # (either sign)
        got = codes[slots[real]]
        assert np.array_equal(np.where(nan[real], got & 0x7F, got), np.where(nan[real], 0x7F, want[real]))
        assert (codes[other] == fill).all() and (exps[other] == fill).all()


def _rows(rng, tokens, width, dtype):
    size = 2.0 ** rng.uniform(-12, 6, (tokens, 1))
    return P.to_bits(rng.standard_normal((tokens, width)) * size, dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hkv,d", [(2, 64), (2, 128), (8, 128), (1, 32), (3, 96), (1, 160), (2, 192), (1, 224), (5, 256)])
@pytest.mark.parametrize("tokens,block", [(1, 16), (37, 48)])
def test_rows_are_written(tokens, block, hkv, d, dtype):
    rng = np.random.default_rng(tokens + d)
    x = _rows(rng, tokens, 2 * hkv * d, dtype)
    pools = Pools(tokens // block + 3, block, hkv, d)
    _check_write(x, hkv, d, _slots(rng, tokens, pools.shape[0] * block), pools, dtype)


@pytest.mark.parametrize("tokens", [1023, 2049, 5000, 17000])
def test_many_rows_out_of_wider_ones(tokens):
    rng = np.random.default_rng(tokens)
    x = _rows(rng, tokens, 8 + 2 * 2 * 64 + 24, "bf16")
    pools = Pools(tokens // 32 + 2, 32, 2, 64)
    _check_write(x, 2, 64, _slots(rng, tokens, pools.shape[0] * 32), pools, "bf16", offset=8)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_at_the_ends_of_the_ranges(dtype):
    """Zeros, the smallest and largest values of the type, maxima next to where the exponent changes, ties."""
    big = 65504.0 if dtype == "fp16" else 3.3e38
    small = 2.0 ** -24 if dtype == "fp16" else 2.0 ** -133
    rows = [[0.0], [-0.0], [big, -big, 1.0], [small, -small], [448.0, 1.0, -17.0, 18.0, 19.0, 2.0 ** -6, 2.0 ** -9,
            2.0 ** -10, 3 * 2.0 ** -10], [1.75], [1.7578125], [1.875, 1.0625, 1.1875], [2.0 ** -14, 2.0 ** -20],
            [np.inf, 3.0, -0.5], [-np.inf, np.nan, 2.0], [np.nan], [7.0, np.inf, np.nan, -np.inf]]
    if dtype == "bf16":
        rows += [[2.0 ** -56, 2.0 ** -62], [2.0 ** -60, 2.0 ** -72, 2.0 ** -73, 2.0 ** -74], [2.0 ** 40, 2.0 ** 41],
                 [1.75 * 2.0 ** 40, 2.0 ** 60, -2.0 ** 100], [2.0 ** -130]]
    x = np.zeros((len(rows), 64))
    for i, r in enumerate(rows):
        x[i, 5:5 + len(r)] = r
    bits = P.to_bits(np.concatenate([x, x[::-1]], 1), dtype)
    pools = Pools(2, 16, 1, 64)
    _check_write(bits, 1, 64, np.arange(len(rows), dtype=np.int64) + 3, pools, dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "f32"])
@pytest.mark.parametrize("hkv,d", [(2, 64), (8, 128), (1, 32), (3, 96), (1, 160), (1, 256)])
@pytest.mark.parametrize("tokens", [1, 40, 4500])
def test_rows_are_read_back(tokens, hkv, d, dtype):
    rng = np.random.default_rng(tokens + d)
    block, blocks, pad = 16, 20, 8
    n = block * blocks
    codes = [rng.integers(0, 256, (blocks, block, hkv, d)).astype(np.uint8) for _ in range(2)]  # NaNs among them
    exps = [rng.integers(127 - 40, 127 + 33, (blocks, hkv, block)).astype(np.uint8) for _ in range(2)]
    slots = rng.integers(0, n, tokens)  # (rows named more than once)
    slots[rng.random(tokens) < 0.1] = rng.choice([-1, n, 1 << 40])
    up = hip.DeviceBuffer.from_numpy
    size = P.storage(dtype)().itemsize
    out = [hip.DeviceBuffer((tokens + 1) * (hkv * d + pad) * size) for _ in range(2)]
    for o in out:
        o.fill(0xFF)
    bufs = [up(a) for a in (codes[0], exps[0], codes[1], exps[1], slots)]
    kernels.launch_kv_gather_e4m3(*bufs, *out, tokens, hkv, d, block, blocks, hkv * d + pad, hkv * d + pad, dtype)
    hip.synchronize()
    real = (slots >= 0) & (slots < n)
    for c, e, o in zip(codes, exps, out):
        got = o.to_numpy(P.storage(dtype), (tokens + 1, hkv * d + pad))
        assert (got[:, hkv * d:].view(np.uint8) == 0xFF).all() and (got[-1].view(np.uint8) == 0xFF).all()
        rows = R.dequantise(c.reshape(n, hkv, d), e.transpose(0, 2, 1).reshape(n, hkv).astype(np.int64) - 127)
        want = np.zeros((tokens, hkv * d))
        want[real] = rows[slots[real]].reshape(-1, hkv * d)
        got = got[:tokens, :hkv * d]
        if dtype == "fp16":
            want = want.clip(-65504, 65504)
        nan = np.isnan(want)
        back = P.from_bits(got, dtype)
        assert np.isnan(back[nan]).all()
        with np.errstate(all="ignore"):
            want = P.from_bits(P.to_bits(want, dtype), dtype)  # (exact but for fp16's rounding)
        assert np.array_equal(back[~nan], want[~nan])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_row_comes_back_within_half_a_step(dtype):
    rng = np.random.default_rng(9)
    tokens, hkv, d = 300, 2, 128
    x = _rows(rng, tokens, 2 * hkv * d, dtype)
    pools = Pools(20, 16, hkv, d)
    slots = rng.permutation(320)[:tokens].astype(np.int64)
    _write(x, hkv, d, slots, pools, dtype)
    out = [hip.DeviceBuffer(tokens * hkv * d * 4) for _ in range(2)]
    at = hip.DeviceBuffer.from_numpy(slots)
    kernels.launch_kv_gather_e4m3(pools.k, pools.k_exp, pools.v, pools.v_exp, at, *out, tokens, hkv, d, 16, 20, dtype="f32")
    hip.synchronize()
    for which, o in enumerate(out):
        want = P.from_bits(x[:, which * hkv * d:(which + 1) * hkv * d], dtype).reshape(tokens, hkv, d)
        got = o.to_numpy(np.float32, (tokens, hkv, d)).astype(np.float64)
        e = R.quantise(want)[1]
        P.assert_within(got, want, np.maximum(np.abs(want) * 2.0 ** -4, (2.0 ** (e - 10.0))[..., None]))


def test_far_rows():
    """Slots whose bytes lie beyond 2^32."""
    hkv, d, block = 64, 256, 1024
    blocks = (1 << 32) // (hkv * d * block) + 3
    rng = np.random.default_rng(4)
    x = _rows(rng, 3, 2 * hkv * d, "bf16")
    slots = np.array([5, (blocks - 2) * block + 7, blocks * block - 1], np.int64)
    rows, at = hip.DeviceBuffer.from_numpy(x), hip.DeviceBuffer.from_numpy(slots)
    k, v = (hip.DeviceBuffer(blocks * block * hkv * d) for _ in range(2))
    k_exp, v_exp = (hip.DeviceBuffer(blocks * block * hkv) for _ in range(2))
    out = [hip.DeviceBuffer(3 * hkv * d * 4) for _ in range(2)]
    kernels.launch_kv_write_e4m3(rows, rows.offset(2 * hkv * d), k, k_exp, v, v_exp, at, 3, hkv, d, block, blocks,
                                 2 * hkv * d, 2 * hkv * d, True)
    kernels.launch_kv_gather_e4m3(k, k_exp, v, v_exp, at, *out, 3, hkv, d, block, blocks, dtype="f32")
    hip.synchronize()
    for which, o in enumerate(out):
        want = R.dequantise(*R.quantise(P.from_bits(x[:, which * hkv * d:(which + 1) * hkv * d], "bf16").reshape(3, hkv, d)))
        assert np.array_equal(o.to_numpy(np.float32, want.shape), want)
