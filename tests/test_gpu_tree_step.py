"""One layer's attention half of a verification step, as a program runs it: norms and positions of the drafted rows,
K and V into the e4m3 cache, attention over it, a prefix read back; launch by launch and captured into a graph."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as P
from tests import tree_reference as R
from tests.test_gpu_paged_attn_tree import random_parents

pytestmark = pytest.mark.gpu


class Step:
    """Sequences with a written context, `new[s]` drafted rows behind it, fused q/k/v rows of the drafted tokens."""

    def __init__(self, seed, new, prior, hq, hkv, d, dtype, block=16):
        rng = np.random.default_rng(seed)
        self.__dict__.update(new=new, prior=prior, hq=hq, hkv=hkv, d=d, dtype=dtype, block=block)
        self.T, self.S = sum(new), len(new)
        self.ctx = np.array(new) + np.array(prior)
        blocks = -(-self.ctx // block)
        self.num_blocks = int(blocks.sum()) + 1
        self.table = np.full((self.S, int(blocks.max())), 0x3FFFFFFF, np.int32)
        ids = rng.permutation(self.num_blocks)
        for s, n in enumerate(blocks):
            self.table[s, :n] = ids[blocks[:s].sum():blocks[:s].sum() + n]
        self.parents = [random_parents(rng, n) for n in new]
        mask = np.concatenate([kernels.tree_mask(p, 1) for p in self.parents])
        depth = [R.ancestors(p).sum(1) - 1 for p in self.parents]
        # a drafted token's position is that of its depth behind the context, on every axis here
        at = np.concatenate([np.array(p) + dep for p, dep in zip(prior, depth)]).astype(np.int32)
        self.positions = np.stack([at, at // 2])
        self.axis = (np.arange(d // 2) % 2).astype(np.uint8)
        self.freq = kernels.rope_frequencies(d, 1e6)[0]
        self.gains = rng.uniform(0.5, 2, (2, d)).astype(np.float32)
        self.rows = P.to_bits(rng.standard_normal((self.T, (hq + 2 * hkv) * d)), dtype)
        self.context = P.to_bits(rng.standard_normal((sum(prior), 2 * hkv * d)), dtype)
        up = hip.DeviceBuffer.from_numpy
        self.b = dict(rows=up(self.rows), positions=up(self.positions), axis=up(self.axis), freq=up(self.freq),
                      gains=up(self.gains), table=up(self.table), mask=up(mask), context=up(self.context),
                      new=up(np.array(new, np.int32)), prior=up(np.array(prior, np.int32)))
        rows = self.num_blocks * block
        for name, size in dict(k=rows * hkv * d, v=rows * hkv * d, k_exp=rows * hkv, v_exp=rows * hkv,
                               cu=4 * (self.S + 1), slots=8 * self.T, ctx=4 * self.S, prefix=8 * sum(prior),
                               none=4 * self.S, cu0=4 * (self.S + 1), ctx0=4 * self.S, q=2 * self.T * hq * d,
                               knew=2 * self.T * hkv * d, out=2 * self.T * hq * d,
                               back_k=2 * sum(prior) * hkv * d, back_v=2 * sum(prior) * hkv * d,
                               ws=kernels.paged_attn_tree_workspace_bytes(self.T, max(new), hq, hkv, d)).items():
            self.b[name] = hip.DeviceBuffer(size)
            self.b[name].fill(0 if name == "none" else 0xFF)
        # the context is in the cache before the step
        kernels.launch_pack_ragged(self.b["prior"], self.b["none"], self.b["table"], self.b["cu0"], self.b["prefix"],
                                   self.b["ctx0"], self.S, block, self.table.shape[1])
        self.write(self.b["context"], self.b["context"].offset(2 * hkv * d), self.b["prefix"], sum(prior), 2 * hkv * d,
                   2 * hkv * d)
        hip.synchronize()

    def write(self, k, v, slots, tokens, ks, vs, stream=None):
        b = self.b
        kernels.launch_kv_write_e4m3(k, v, b["k"], b["k_exp"], b["v"], b["v_exp"], slots, tokens, self.hkv, self.d,
                                     self.block, self.num_blocks, ks, vs, self.dtype == "bf16", stream)

    def launch(self, stream=None):
        b, hq, hkv, d = self.b, self.hq, self.hkv, self.d
        width = (hq + 2 * hkv) * d
        kernels.launch_pack_ragged(b["new"], b["prior"], b["table"], b["cu"], b["slots"], b["ctx"], self.S, self.block,
                                   self.table.shape[1], stream)
        kernels.launch_norm_rope_packed(b["rows"], b["rows"].offset(2 * hq * d), b["q"], b["knew"], b["positions"], b["axis"],
                                        b["freq"], b["gains"], b["gains"].offset(4 * d), self.T, hq, hkv, d, d, num_axes=2,
                                        q_in_stride=width, k_in_stride=width, dtype=self.dtype, stream=stream)
        self.write(b["knew"], b["rows"].offset(2 * (hq + hkv) * d), b["slots"], self.T, hkv * d, width, stream)
        kernels.launch_paged_attn_tree(b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"], b["mask"], b["out"], b["ws"],
                                       self.S, self.T, max(self.new), hq, hkv, d, self.block, self.table.shape[1],
                                       self.num_blocks, 1 / np.sqrt(d), 1, b["k_exp"], b["v_exp"], bf16=self.dtype == "bf16",
                                       stream=stream)
        kernels.launch_kv_gather_e4m3(b["k"], b["k_exp"], b["v"], b["v_exp"], b["prefix"], b["back_k"], b["back_v"],
                                      sum(self.prior), hkv, d, self.block, self.num_blocks, dtype=self.dtype, stream=stream)

    def results(self):
        hip.synchronize()
        t = P.storage(self.dtype)
        shapes = dict(q=(self.T, self.hq, self.d), knew=(self.T, self.hkv, self.d), out=(self.T, self.hq, self.d),
                      back_k=(sum(self.prior), self.hkv, self.d), back_v=(sum(self.prior), self.hkv, self.d))
        return {n: self.b[n].to_numpy(t, s) for n, s in shapes.items()}

    def check(self, got):
        """Every operator against the 64-bit form of what it was given."""
        hq, hkv, d = self.hq, self.hkv, self.d
        val = lambda a: P.from_bits(a, self.dtype)  # noqa: E731
        x = val(self.rows).reshape(self.T, hq + 2 * hkv, d)
        for name, at, gain in (("q", slice(0, hq), 0), ("knew", slice(hq, hq + hkv), 1)):
            want, bound = R.norm_rope(x[:, at], self.gains[gain].astype(np.float64), 1e-6, self.positions, self.axis, self.freq,
                                      d, False, 1.0, self.dtype)
            P.assert_within(val(got[name]), want, bound, name)
        old = val(self.context).reshape(-1, 2, hkv, d)
        new = np.stack([val(got["knew"]), x[:, hq + hkv:]], 1)
        t0 = c0 = 0
        for s in range(self.S):
            n, c = self.new[s], self.prior[s]
            rows = np.concatenate([old[c0:c0 + c], new[t0:t0 + n]])
            (kc, ke), (vc, ve) = R.quantise(rows[:, 0]), R.quantise(rows[:, 1])
            k, v = R.dequantise(kc, ke), R.dequantise(vc, ve)
            for name, r in (("back_k", k), ("back_v", v)):
                assert np.array_equal(val(got[name][c0:c0 + c]), val(P.to_bits(r[:c], self.dtype)))
            if n:
                seen = np.ones((n, c + n), bool)
                seen[:, c:] = R.ancestors(self.parents[s])
                want, bound = R.tree_attention(val(got["q"][t0:t0 + n]), k, v, seen, 1 / np.sqrt(d), self.dtype, ke, ve)
                P.assert_within(val(got["out"][t0:t0 + n]), want, bound, f"sequence {s}")
            t0, c0 = t0 + n, c0 + c


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (14, 2, 64)])
def test_a_step(hq, hkv, d, dtype):
    s = Step(1, [9, 1, 30, 0], [100, 515, 16, 40], hq, hkv, d, dtype)
    s.launch()
    s.check(s.results())


def test_a_captured_step_replays():
    s = Step(2, [8, 21, 3], [700, 33, 250], 12, 2, 128, "bf16")
    s.launch()
    want = s.results()
    stream = hip.Stream()
    graph = hip.Graph(stream)
    with graph:
        s.launch(stream)
    for _ in range(4):
        for name in ("q", "knew", "out", "back_k", "back_v", "cu", "slots", "ctx", "ws"):
            s.b[name].fill(0xFF)
        hip.synchronize()
        graph.launch()
        stream.synchronize()
        got = s.results()
        assert all(np.array_equal(got[n], want[n]) for n in want)
        s.launch()  # the program's own calls between the replays
        assert np.array_equal(s.results()["out"], want["out"])
    s.check(want)
