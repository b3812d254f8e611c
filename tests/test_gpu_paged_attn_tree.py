"""Attention of drafted tokens over fp16 and e4m3 pools, against the 64-bit form."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as P
from tests import tree_reference as R

pytestmark = pytest.mark.gpu

KINDS = [("fp16", "fp16"), ("e4m3", "fp16"), ("e4m3", "bf16")]  # pools, rows


def random_parents(rng, n):
    return np.array([-1 if i == 0 or rng.random() < 0.05 else rng.integers(max(0, i - 9), i) for i in range(n)], int)


class Case:
    """Sequences of new[s] drafted rows behind prior[s] rows of context, in pools of scattered blocks; seen[s] bool
    [n][n] (None: random trees)."""

    def __init__(self, seed, new, prior, hq, hkv, d, pool="fp16", dtype="fp16", block=16, words=None, seen=None, pad=0,
                 front=0, behind=0, scale=None):
        rng = np.random.default_rng(seed)
        self.__dict__.update(hq=hq, hkv=hkv, d=d, pool=pool, dtype=dtype, block=block, pad=pad)
        self.new, self.ctx = np.array(new), np.array(new) + np.array(prior)
        self.scale = 1 / np.sqrt(d) if scale is None else scale
        self.cu = front + np.concatenate([[0], np.cumsum(self.new)])
        self.total = int(self.cu[-1]) + behind
        self.seen = seen or [R.ancestors(random_parents(rng, n)) for n in new]
        self.words = words or max(1, (max(new) + 63) // 64)
        self.mask = np.zeros((self.total, self.words), np.uint64)
        for s, m in enumerate(self.seen):
            if new[s]:
                self.mask[self.cu[s]:self.cu[s + 1]] = R.mask_bits(np.asarray(m), self.words)
        blocks = -(-self.ctx // block)
        self.num_blocks = int(blocks.sum()) + 2
        self.table = np.full((len(new), max(1, int(blocks.max())) + 1), 0x3FFFFFFF, np.int32)
        ids = rng.permutation(self.num_blocks - 1)[:int(blocks.sum())] + 1  # (block 0 is nobody's)
        for s, n in enumerate(blocks):
            self.table[s, :n] = ids[blocks[:s].sum():blocks[:s].sum() + n]
        self.q = P.to_bits(rng.standard_normal((self.total, hq * d + pad)), dtype)
        self.set_rows(*(rng.standard_normal((self.num_blocks, block, hkv, d), np.float32).astype(np.float16)
                        for _ in range(2)))

    def set_rows(self, k, v):
        self.k16, self.v16 = k, v
        if self.pool == "fp16":
            self.k, self.v, self.k_exp, self.v_exp = k, v, None, None
        else:
            (self.k, ke), (self.v, ve) = (R.quantise(x.astype(np.float64)) for x in (k, v))
            self.k_exp, self.v_exp = ((e + 127).astype(np.uint8).transpose(0, 2, 1).copy() for e in (ke, ve))

    def values(self, s):
        """K, V and exponents of sequence s in order."""
        c, ids = int(self.ctx[s]), self.table[s, :-(-int(self.ctx[s]) // self.block)]
        out = []
        for pool, exp in ((self.k, self.k_exp), (self.v, self.v_exp)):
            if exp is None:
                out.append((pool[ids].reshape(-1, self.hkv, self.d)[:c].astype(np.float64), None))
            else:
                e = exp[ids].transpose(0, 2, 1).reshape(-1, self.hkv)[:c].astype(np.int64) - 127
                out.append((R.dequantise(pool[ids].reshape(-1, self.hkv, self.d)[:c], e), e))
        return out

    def visible(self, s):
        n, c = int(self.new[s]), int(self.ctx[s])
        seen = np.ones((n, c), bool)
        seen[:, c - n:] = np.asarray(self.seen[s])[:, :n]
        for j, b in enumerate(self.table[s, :-(-c // self.block)]):
            if not 0 <= b < self.num_blocks:
                seen[:, j * self.block:(j + 1) * self.block] = False
        return seen

    def want(self, s):
        (k, ke), (v, ve) = self.values(s)
        q = P.from_bits(self.q[self.cu[s]:self.cu[s + 1], :self.hq * self.d], self.dtype)
        return R.tree_attention(q.reshape(-1, self.hq, self.d), k, v, self.visible(s), self.scale, self.dtype, ke, ve)

    def upload(self):
        up = hip.DeviceBuffer.from_numpy
        self.bufs = dict(q=up(self.q), k=up(self.k), v=up(self.v), table=up(self.table), cu=up(self.cu.astype(np.int32)),
                         ctx=up(self.ctx.astype(np.int32)), mask=up(self.mask))
        if self.k_exp is not None:
            self.bufs.update(k_exp=up(self.k_exp), v_exp=up(self.v_exp))
        self.bufs["out"] = hip.DeviceBuffer(self.q.nbytes)
        self.bufs["out"].fill(0xFF)
        ws = kernels.paged_attn_tree_workspace_bytes(self.total, self.longest, self.hq, self.hkv, self.d)
        self.bufs["ws"] = hip.DeviceBuffer(ws)
        self.bufs["ws"].fill(0xFF)

    @property
    def longest(self):
        return max(1, int(self.new.max()))

    def launch(self, stream=None, ws=None, out=None):
        b = self.bufs
        kernels.launch_paged_attn_tree(
            b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"], b["mask"], out or b["out"], ws or b["ws"],
            len(self.new), self.total, self.longest, self.hq, self.hkv, self.d, self.block, self.table.shape[1],
            self.num_blocks, float(self.scale), self.words, b.get("k_exp"), b.get("v_exp"), self.q.shape[1],
            self.q.shape[1], self.dtype == "bf16", stream)

    def run(self):
        self.upload()
        self.launch()
        hip.synchronize()
        return self.bufs["out"].to_numpy(self.q.dtype, self.q.shape)

    def check(self, sequences=None):
        out = self.run()
        w = self.hq * self.d
        assert (out[:, w:].view(np.uint8) == 0xFF).all()
        for rows in (slice(0, self.cu[0]), slice(self.cu[-1], None)):
            assert (out[rows].view(np.uint8) == 0xFF).all()
        for s in range(len(self.new)) if sequences is None else sequences:
            if self.new[s]:
                want, bound = self.want(s)
                got = P.from_bits(out[self.cu[s]:self.cu[s + 1], :w], self.dtype).reshape(want.shape)
                P.assert_within(got, want, bound, f"sequence {s}")
        return out


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128), (32, 8, 128), (8, 1, 128), (16, 16, 96), (8, 1, 256),
                                      (24, 4, 32), (10, 2, 160), (2, 1, 192), (3, 1, 224), (40, 1, 64)])
def test_geometries(hq, hkv, d, pool, dtype):
    Case(1, [7, 1, 0, 20], [300, 77, 50, 0], hq, hkv, d, pool, dtype).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("prior", [0, 1, 8, 15, 16, 17, 24, 31, 32, 33, 63, 64, 100, 1000, 5003])
@pytest.mark.parametrize("n", [1, 5, 33, 64])
def test_contexts(n, prior, pool, dtype):
    Case(n + prior, [n], [prior], 6, 2, 64, pool, dtype, block=48 if prior % 2 else 16).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("n,words", [(65, 2), (100, 4), (128, 2), (200, 4), (256, 4)])
def test_many_drafted_tokens(n, words, pool, dtype):
    Case(n, [n, 3], [70, 500], 8, 2, 64, pool, dtype, words=words).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (14, 2, 64), (4, 4, 32)])
def test_contexts_that_are_cut(hq, hkv, d, pool, dtype):
    """Few sequences and many keys: units shared by many workgroups, workgroups with the end of one and the beginning
    of the next."""
    Case(3, [9, 2, 30], [20000, 33, 9001], hq, hkv, d, pool, dtype, block=64).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
def test_many_sequences(pool, dtype):
    rng = np.random.default_rng(5)
    new = rng.integers(0, 4, 150)
    new[[3, 70, 149]] = 17, 0, 12
    c = Case(6, new.tolist(), rng.integers(0, 200, 150).tolist(), 4, 2, 64, pool, dtype, front=3, behind=5)
    c.check()


@pytest.mark.parametrize("pool,dtype", KINDS)
def test_strides_and_rows_that_are_not_there(pool, dtype):
    Case(7, [4, 6], [40, 5], 4, 2, 96, pool, dtype, pad=40, front=7, behind=2).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
def test_any_masks(pool, dtype):
    """Rows that see none of the new tokens, not themselves, tokens behind them, all of them; no key at all."""
    rng = np.random.default_rng(8)
    seen = [rng.random((40, 40)) < 0.3, np.ones((33, 33), bool), np.zeros((10, 10), bool), np.zeros((5, 5), bool)]
    seen[0][::7] = False
    c = Case(9, [40, 33, 10, 5], [100, 0, 64, 0], 6, 2, 64, pool, dtype, seen=seen)
    out = c.check()
    assert not out[c.cu[3]:].any()  # nothing to see: zeros


def test_bits_behind_the_last_token_are_not_looked_at():
    c = Case(10, [5, 20], [50, 3], 4, 2, 64, words=2)
    want = c.run()
    for s in range(2):
        n = int(c.new[s])
        c.mask[c.cu[s]:c.cu[s + 1], 0] |= np.uint64((~((1 << n) - 1)) & (2 ** 64 - 1))
        c.mask[c.cu[s]:c.cu[s + 1], 1] = np.uint64(2 ** 64 - 1)
    assert np.array_equal(c.run(), want)


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_seen_does_not_matter(bad, pool, dtype):
    """Infinities and NaN in rows of the pools that a token does not see: behind the last, in blocks of nobody, in K and V of
    other branches.  Tokens that see them are as they come; the others are what they are without."""
    c = Case(11, [12, 30, 64], [37, 160, 300], 6, 2, 64, pool, dtype)
    clean = c.run()
    within = [c.want(s) for s in range(3)]
    free = np.ones((c.num_blocks, c.block), bool)
    hit = []
    for s in range(3):
        ctx, n = int(c.ctx[s]), int(c.new[s])
        for j in range(ctx):
            free[c.table[s, j // c.block], j % c.block] = False
        hit.append(n // 2)
    k, v = c.k16.copy(), c.v16.copy()
    k[free], v[free] = bad, bad
    for s, j in enumerate(hit):
        at = int(c.ctx[s] - c.new[s]) + j
        b = c.table[s, at // c.block], at % c.block
        v[b][:, ::3] = bad
        if s != 1:
            k[b][:, 1::2] = bad
    c.set_rows(k, v)
    out = c.run()
    for s, j in enumerate(hit):
        sees = np.asarray(c.seen[s])[:, j]
        rows = np.arange(c.cu[s], c.cu[s + 1])
        if pool == "fp16":
            assert np.array_equal(out[rows[~sees]], clean[rows[~sees]])
        # (e4m3: the exponents that 32 neighbours are taken relative to may have changed)
        P.assert_within(P.from_bits(out[rows], dtype).reshape(within[s][0].shape)[~sees], *(w[~sees] for w in within[s]))
        got = P.from_bits(out[rows[sees]], dtype).reshape(-1, c.hq, c.d)
        assert sees.any() and (~np.isfinite(got[..., ::3])).all()
        if s == 1 and pool == "fp16":  # V alone: an infinity stays one, and in its elements
            assert np.isfinite(got[..., 1::3]).all()
            assert (np.isnan(got[..., ::3]) if np.isnan(bad) else got[..., ::3] == bad).all()


@pytest.mark.parametrize("pool,dtype", KINDS)
def test_blocks_that_are_none(pool, dtype):
    """A table entry outside the pools hides its keys, in the context and among the new tokens."""
    for block in (16, 48):
        c = Case(12, [20, 3, 6], [300, 100, 17], 6, 2, 64, pool, dtype, block=block)
        c.table[0, 2] = -1
        c.table[0, -2] = c.num_blocks
        c.table[1, 0] = 0x3FFFFFFF
        c.table[2, :] = -(1 << 31)
        out = c.run()
        for s in (0, 1):
            k, v = c.values_of_real_blocks(s)
            q = P.from_bits(c.q[c.cu[s]:c.cu[s + 1]], dtype).reshape(-1, c.hq, c.d)
            want, bound = R.tree_attention(q, k[0], v[0], c.visible(s), c.scale, dtype, k[1], v[1])
            P.assert_within(P.from_bits(out[c.cu[s]:c.cu[s + 1]], dtype).reshape(want.shape), want, bound)
        assert not out[c.cu[2]:].any()


def _real_blocks(self, s):
    table = self.table.copy()
    self.table = np.where((table >= 0) & (table < self.num_blocks), table, 0).astype(np.int32)
    try:
        return self.values(s)
    finally:
        self.table = table


Case.values_of_real_blocks = _real_blocks


@pytest.mark.parametrize("pool,dtype", KINDS)
def test_rows_of_very_different_sizes(pool, dtype):
    """K and V rows from 2^-8 to 2^8 of one another, also between neighbours; scores up to some hundreds."""
    c = Case(13, [16, 8], [500, 1500], 6, 2, 64, pool, dtype)
    rng = np.random.default_rng(14)
    for name in ("k16", "v16"):
        z = 2.0 ** rng.uniform(-8, 4 if name == "k16" else 8, c.k16.shape[:3])
        setattr(c, name, (getattr(c, name) * z[..., None]).astype(np.float16))
    c.set_rows(c.k16, c.v16)
    c.check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("scale", [1e-6, 3.0, 100.0, 1e5])
def test_scales(scale, pool, dtype):
    """From equal weights to one key that has all of it."""
    Case(15, [10, 3], [400, 40], 6, 2, 64, pool, dtype, scale=scale).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("shift", [10, 19, 20, 21, 23, 24, 26, 27, 28, 29, 40, 100])
def test_scores_far_apart(shift, pool, dtype):
    """Whole numbers as scores, times 2^shift: the keys with the largest share all the weight."""
    c = Case(30 + shift, [9, 40], [300, 70], 6, 2, 64, pool, dtype, scale=2.0 ** shift)
    rng = np.random.default_rng(31)
    c.q = P.to_bits(rng.integers(-1, 2, c.q.shape), dtype)
    c.set_rows(rng.integers(-1, 2, c.k16.shape).astype(np.float16), c.v16)
    out = c.run()
    for s in range(2):
        (k, _), (v, ve) = c.values(s)
        q = P.from_bits(c.q[c.cu[s]:c.cu[s + 1]], dtype).reshape(-1, c.hq, c.d)
        got = P.from_bits(out[c.cu[s]:c.cu[s + 1]], dtype).reshape(q.shape)
        seen = c.visible(s)
        for h in range(c.hq):
            score = np.where(seen, q[:, h] @ k[:, h // 3].T, -np.inf)
            w = (score == score.max(1, keepdims=True)).astype(float)
            w /= w.sum(1, keepdims=True)
            want, size = w @ v[:, h // 3], w @ np.abs(v[:, h // 3])
            # equal weights, off by half a step of fp16 and by fp32 sums; of neighbours' rows of V 2^-25 of the largest step
            bound = (2.0 ** -11 + 2.0 ** -16) * size + 2.0 ** -24 * np.abs(v).max() + P.HALF_STEP[dtype] * np.abs(want) + 2.0 ** -25
            P.assert_within(got[:, h], want, bound)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_small_exponents(dtype):
    """Rows near the lowest numbers of fp16 beside ordinary ones, one of them with all the weight."""
    c = Case(16, [4], [90], 4, 2, 64, "e4m3", dtype)
    rng = np.random.default_rng(17)
    c.v16 = (rng.standard_normal(c.v16.shape) * 2.0 ** -20).astype(np.float16)
    c.set_rows(c.k16, c.v16)
    c.check()


def test_one_new_token_is_the_decode_step():
    """What the paged attention gives for one new token per sequence, to its bound."""
    rng = np.random.default_rng(18)
    prior = rng.integers(1, 700, 9).tolist()
    c = Case(19, [1] * 9, prior, 12, 2, 128)
    mine = c.check()
    splits = kernels.paged_attn_num_splits(9, 2, 16, c.table.shape[1], 128)
    ws = hip.DeviceBuffer(max(16, kernels.paged_attn_workspace_bytes(9, 12, 128, splits)))
    out = hip.DeviceBuffer(c.q.nbytes)
    b = c.bufs
    kernels.launch_paged_attn_varlen_fp16(b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"], out, ws, 9, 9, 1, 12, 2, 128,
                                          16, c.table.shape[1], splits, float(c.scale), True, None)
    hip.synchronize()
    theirs = out.to_numpy(np.float16, c.q.shape)
    for s in range(9):
        want, bound = c.want(s)
        got = theirs[s].astype(np.float64).reshape(want.shape)
        P.assert_within(got, mine[s].astype(np.float64).reshape(want.shape), 2 * bound)


def test_a_chain_is_the_causal_chunk():
    """Masks of bits 0 .. i: what the paged attention gives for a chunk, to its bound."""
    c = Case(20, [40, 9], [100, 0], 12, 2, 128, seen=[np.tri(40, dtype=bool), np.tri(9, dtype=bool)])
    mine = c.check()
    splits = kernels.paged_attn_num_splits(2, 2, 16, c.table.shape[1], 128)
    ws = hip.DeviceBuffer(max(16, kernels.paged_attn_workspace_bytes(2, 12, 128, splits)))
    out = hip.DeviceBuffer(c.q.nbytes)
    b = c.bufs
    kernels.launch_paged_attn_varlen_fp16(b["q"], b["k"], b["v"], b["table"], b["cu"], b["ctx"], out, ws, 2, c.total, 40, 12,
                                          2, 128, 16, c.table.shape[1], splits, float(c.scale), True, None)
    hip.synchronize()
    theirs = out.to_numpy(np.float16, c.q.shape).astype(np.float64)
    for s in range(2):
        want, bound = c.want(s)
        rows = slice(c.cu[s], c.cu[s + 1])
        P.assert_within(theirs[rows].reshape(want.shape), mine[rows].astype(np.float64).reshape(want.shape), 2 * bound)


def test_far_blocks():
    """Blocks whose bytes lie beyond 2^32."""
    hkv, d, block = 16, 256, 4096
    c = Case(21, [3], [40], 16, hkv, d)
    blocks = (1 << 32) // (hkv * d * 2 * block) + 2
    far = np.array([[blocks - 1]], np.int32)
    rows = [np.zeros((block, hkv, d), np.float16) for _ in range(2)]
    for r, (x, _) in zip(rows, c.values(0)):
        r[:len(x)] = x
    pools = []
    for r in rows:
        pool = hip.DeviceBuffer(blocks * r.nbytes)
        one = hip.DeviceBuffer.from_numpy(r)
        pool.copy_from_device(one, r.nbytes, (blocks - 1) * r.nbytes)
        pools.append(pool)
    want, bound = c.want(0)
    c.upload()
    c.bufs.update(k=pools[0], v=pools[1], table=hip.DeviceBuffer.from_numpy(far))
    c.block, c.num_blocks, c.table = block, blocks, far
    c.launch()
    hip.synchronize()
    got = c.bufs["out"].to_numpy(np.float16, c.q.shape).astype(np.float64).reshape(want.shape)
    P.assert_within(got, want, bound)


def test_two_calls_at_once_and_the_same_bits_every_time():
    """Two streams with a workspace each, beside one another; every result as it is alone."""
    cases = [Case(22, [9, 4], [9000, 50], 12, 2, 128), Case(23, [5] * 6, [700] * 6, 8, 2, 64, "e4m3", "bf16")]
    want = [c.run() for c in cases]
    streams = [hip.Stream(), hip.Stream()]
    for _ in range(5):
        for c, s in zip(cases, streams):
            c.bufs["out"].fill(0xFF)
            hip.synchronize()
        for _ in range(3):
            for c, s in zip(cases, streams):
                c.launch(s)
        hip.synchronize()
        for c, w in zip(cases, want):
            assert np.array_equal(c.bufs["out"].to_numpy(c.q.dtype, c.q.shape), w)


def test_a_captured_call_replays_with_other_contexts():
    """The lengths are the device's: a captured call serves the steps that follow."""
    c = Case(24, [6, 1, 11], [800, 300, 40], 6, 2, 64, "e4m3", "fp16")
    c.upload()
    stream = hip.Stream()
    graph = hip.Graph(stream)
    with graph:
        c.launch(stream)
    for prior in ([800, 300, 40], [20, 301, 0], [700, 0, 5]):
        c.ctx = np.array(prior) + c.new
        ctx = hip.DeviceBuffer.from_numpy(c.ctx.astype(np.int32))
        c.bufs["ctx"].copy_from_device(ctx, ctx.nbytes)
        c.bufs["out"].fill(0xFF)
        c.bufs["ws"].fill(0xFF)
        hip.synchronize()
        graph.launch()
        stream.synchronize()
        out = c.bufs["out"].to_numpy(c.q.dtype, c.q.shape)
        for s in range(3):
            want, bound = c.want(s)
            P.assert_within(P.from_bits(out[c.cu[s]:c.cu[s + 1]], c.dtype).reshape(want.shape), want, bound)
        other = hip.DeviceBuffer(c.q.nbytes)
        c.launch(out=other)
        hip.synchronize()
        assert np.array_equal(other.to_numpy(c.q.dtype, c.q.shape), out)
