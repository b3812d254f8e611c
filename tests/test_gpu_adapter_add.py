"""Low-rank adapters beside a shared projection against the 64-bit form."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as R

pytestmark = pytest.mark.gpu

GUARD = 2
NAN = {"fp16": np.float16(np.nan), "bf16": np.uint16(0x7FC0)}


def _case(seed, lens, pick, ranks, max_rank, n, k, dtype, out_dtype=None, pads=(0, 0, 0)):
    rng = np.random.default_rng(seed)
    out_dtype = out_dtype or dtype
    T, A = int(sum(lens)) + GUARD, len(ranks)

    def normal(*shape, dev=1.0, to=dtype):
        return R.to_bits(rng.standard_normal(shape, np.float32) * np.float32(dev), to)

    c = dict(x=normal(T, k + pads[0]), a=normal(A, max_rank, k, dev=k ** -0.5),
             b=normal(A, n, max_rank, dev=0.3), base=normal(T, n + pads[1], to=out_dtype),
             ranks=np.asarray(ranks, np.int32), scales=rng.uniform(0.5, 2, A).astype(np.float32),
             pick=np.asarray(pick, np.int32), lens=list(lens), n=n, k=k, max_rank=max_rank, T=T,
             dtype=dtype, out_dtype=out_dtype, out_stride=n + pads[2])
    for i, r in enumerate(ranks):  # what lies behind an adapter's rank is not looked at
        c["a"][i, max(r, 0):] = NAN[dtype]
        c["b"][i, :, max(r, 0):] = NAN[dtype]
    return c


class Run:
    def __init__(self, c, in_place=False, stream=None):
        self.c, self.stream, self.in_place = c, stream, in_place
        self.buf = {x: hip.DeviceBuffer.from_numpy(c[x])
                    for x in ("x", "a", "b", "base", "ranks", "scales", "pick")}
        self.cu = hip.DeviceBuffer.from_numpy(np.concatenate([[0], np.cumsum(c["lens"])]).astype(np.int32))
        self.stride = c["base"].shape[1] if in_place else c["out_stride"]
        self.out = self.buf["base"] if in_place else \
            hip.DeviceBuffer(c["T"] * self.stride * c["base"].dtype.itemsize)
        if not in_place:
            self.out.fill(0xFF)
        self.ws = hip.DeviceBuffer(kernels.adapter_add_workspace_bytes(c["T"], c["max_rank"]))
        self.ws.fill(0xFF)

    def launch(self):
        c, b = self.c, self.buf
        kernels.launch_adapter_add(
            b["x"], b["a"], b["b"], b["ranks"], b["scales"], b["pick"], self.cu, b["base"], self.out,
            self.ws, len(c["lens"]), c["T"], len(c["ranks"]), c["max_rank"], c["n"], c["k"],
            c["x"].shape[1], c["base"].shape[1], self.stride, bf16=c["dtype"] == "bf16",
            f32_out=c["out_dtype"] == "f32", stream=self.stream)

    def bits(self):
        (self.stream.synchronize() if self.stream else hip.synchronize())
        return self.out.to_numpy(self.c["base"].dtype, (self.c["T"], self.stride))


def _want(c):
    n = sum(c["lens"])
    f = lambda a, t=c["dtype"]: R.from_bits(a, t)  # noqa: E731
    return R.adapter(f(c["x"][:n, :c["k"]]), f(c["a"]), f(c["b"]), c["ranks"], c["scales"], c["pick"],
                     c["lens"], f(c["base"][:n, :c["n"]], c["out_dtype"]), c["dtype"], c["out_dtype"])


def _check(c):
    n = sum(c["lens"])
    want, bound = _want(c)
    r = Run(c)
    r.launch()
    got = r.bits()
    raw = got.view(np.uint8).reshape(c["T"], -1)
    assert (raw[n:] == 0xFF).all() and (raw[:, c["n"] * got.dtype.itemsize:] == 0xFF).all()
    R.assert_within(R.from_bits(got[:n, :c["n"]], c["out_dtype"]), want, bound)
    bare = np.repeat([not 0 <= p < len(c["ranks"]) or c["ranks"][p] <= 0 for p in c["pick"]], c["lens"])
    assert np.array_equal(got[:n, :c["n"]][bare], c["base"][:n, :c["n"]][bare])
    # in place: the same bits, the rest of the rows as they were
    r = Run(c, in_place=True)
    r.launch()
    there = r.bits()
    assert np.array_equal(there[:n, :c["n"]], got[:n, :c["n"]])
    there[:n, :c["n"]] = c["base"][:n, :c["n"]]
    assert np.array_equal(there, c["base"])


OUTS = [("fp16", "fp16"), ("bf16", "bf16"), ("fp16", "f32"), ("bf16", "f32")]


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("ranks,max_rank", [([1], 8), ([8], 8), ([5, 16], 16), ([17, 3, 24], 24),
                                            ([32, 33, 64], 64), ([100, 128], 128), ([256, 200], 256),
                                            ([15, 40], 40)])
def test_ranks(ranks, max_rank, dtype, out):
    A = len(ranks)
    lens = [1, 1, 40, 1, 7, 17]
    _check(_case(1, lens, np.arange(6) % A, ranks, max_rank, 264, 200, dtype, out))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("n,k", [(8, 8), (64, 32), (256, 512), (896, 896), (1032, 4864), (1536, 8960),
                                 (24, 1000), (4104, 40)])
def test_sizes(n, k, dtype, out):
    _check(_case(2, [1, 33, 1, 0, 5], [1, 0, 2, 1, 2], [16, 8, 13], 16, n, k, dtype, out))


@pytest.mark.parametrize("dtype,out", OUTS)
def test_sequences_without_an_adapter(dtype, out):
    _check(_case(3, [1, 20, 1, 3, 1, 64], [-1, 0, 3, 1, -(1 << 31), 2], [16, 0, -5], 16, 136, 256, dtype, out))
    _check(_case(4, [1, 30], [-1, 7], [16], 16, 136, 256, dtype, out))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("pads", [(8, 0, 0), (0, 16, 8), (24, 8, 128)])
def test_strides(pads, dtype, out):
    _check(_case(5, [1, 35, 2], [0, 1, 0], [16, 9], 16, 328, 264, dtype, out, pads))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens", [[1], [0, 1, 0], [15, 16, 17], [31, 32, 33], [63, 64, 65], [400],
                                  [1] * 200, [127, 128, 129, 1]], ids=lambda v: f"{len(v)} of {max(v)}")
def test_lengths(lens, dtype):
    _check(_case(6, lens, np.arange(len(lens)) % 3, [32, 16, 7], 32, 520, 384, dtype))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("lens,max_rank", [([700, 1, 900], 64), ([512] * 5 + [1] * 30, 16)],
                         ids=["64", "16"])
def test_many_rows(lens, max_rank, dtype, out):
    _check(_case(7, lens, np.arange(len(lens)) % 4, [max_rank, 8, max_rank // 2 + 1, 3], max_rank, 776, 1024,
                 dtype, out))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("max_rank", [16, 32, 48, 64, 104])
@pytest.mark.parametrize("n,k", [(1100, 256), (264, 5000)])
def test_many_short_sequences(n, k, max_rank, dtype, out):
    """More tiles than take both products at once."""
    n = n // 8 * 8
    lens = [1, 2, 0, 1] * 90 + [17]
    _check(_case(13, lens, np.arange(len(lens)) % 5 - 1, [max_rank, 7, max_rank - 3, 12], max_rank, n, k, dtype,
                 out))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("max_rank", [8, 16, 32, 40, 64])
@pytest.mark.parametrize("lens", [[1], [16, 1, 3, 33]], ids=str)
def test_few_rows(lens, max_rank, dtype, out):
    _check(_case(14, lens, np.arange(len(lens)) % 3, [max_rank, max_rank - 5, 0], max_rank, 2104, 1096, dtype, out))
    _check(_case(15, lens, np.arange(len(lens)) % 3 - 1, [max_rank, 1], max_rank, 1024, 4096, dtype, out))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("max_rank", [72, 128, 200, 256])
def test_large_ranks_of_long_sequences(max_rank, dtype, out):
    _check(_case(16, [150, 33, 0, 70], [0, 1, 2, 2], [max_rank, 65, 7], max_rank, 392, 520, dtype, out))


@pytest.mark.parametrize("dtype,out", [("fp16", "fp16"), ("bf16", "f32")])
@pytest.mark.parametrize("max_rank", [32, 64, 128, 256])
@pytest.mark.parametrize("lens", [[33] * 64, [1] * 200], ids=["33", "1"])
def test_workgroups_of_several_steps(lens, max_rank, dtype, out):
    """Enough tiles and outputs that a workgroup walks over its slice; the last slice ends inside a step."""
    pick = np.arange(len(lens)) % 4 - 1
    _check(_case(17, lens, pick, [max_rank, max_rank // 2 + 3, 5], max_rank, 11000, 264, dtype, out))


def test_a_rank_above_the_slot_is_the_slots():
    c = _case(8, [20], [0], [16], 16, 136, 128, "fp16")
    want = Run(c)
    want.launch()
    c["ranks"] = np.array([99], np.int32)
    got = Run(c)
    got.launch()
    assert np.array_equal(got.bits().view(np.uint16), want.bits().view(np.uint16))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("size", [1e-6, 3e3])
def test_small_and_large_products(size, dtype):
    """x A^T far from 1 (fp16 could not hold it as it is)."""
    c = _case(9, [1, 40], [0, 1], [16, 12], 16, 264, 512, dtype, "f32")
    c["x"] = R.to_bits(R.from_bits(c["x"], dtype) * (size if dtype == "bf16" else min(size, 1e3)), dtype)
    if size > 1:
        c["a"] = R.to_bits(R.from_bits(c["a"], dtype) * 300, dtype)
    _check(c)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_infinities_and_nan_stay_in_their_row(dtype):
    c = _case(10, [40], [0], [16], 16, 264, 128, dtype, "f32")
    want, bound = _want(c)
    c["x"][3, 7] = NAN[dtype]
    c["x"][20, 9] = np.float16(np.inf) if dtype == "fp16" else np.uint16(0x7F80)
    r = Run(c)
    r.launch()
    got = R.from_bits(r.bits()[:40], "f32")
    keep = np.setdiff1d(np.arange(40), [3, 20])
    R.assert_within(got[keep], want[keep], bound[keep])
    assert np.isnan(got[3]).all() and not np.isfinite(got[20]).any()


def test_an_infinite_sum_is_infinite():
    """One rank that overflows to +inf times positive columns is +inf, not NaN."""
    for dtype in ("fp16", "bf16"):
        c = _case(11, [18], [0], [1], 8, 64, 64, dtype, "f32")
        c["a"][0, 0] = R.to_bits(np.ones(64), dtype)
        c["b"][0, :, 0] = R.to_bits(np.full(64, 0.5), dtype)
        c["x"][5] = R.to_bits(np.ones(64), dtype)
        c["x"][5, 0] = np.float16(np.inf) if dtype == "fp16" else np.uint16(0x7F80)
        r = Run(c)
        r.launch()
        assert np.isposinf(r.bits()[5]).all()


def test_a_captured_call_replays():
    stream = hip.Stream()
    c = _case(12, [1, 50, 1], [0, 1, -1], [16, 24], 24, 520, 1024, "bf16")
    r = Run(c, stream=stream)
    r.launch()
    want = r.bits().copy()
    hip.synchronize()
    graph = hip.Graph(stream)
    with graph:
        r.launch()
    for _ in range(3):
        r.out.fill(0xFF)
        r.ws.fill(0xFF)
        hip.synchronize()
        graph.launch()
        assert np.array_equal(r.bits(), want)
        r.launch()
        assert np.array_equal(r.bits(), want)
