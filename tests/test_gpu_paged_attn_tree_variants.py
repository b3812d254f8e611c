"""Tree attention by the shape of its workgroups: narrow trees (parts of a workgroup take key tiles in turn), wide ones, units that are
cut and units that are not, more tiles than a workgroup keeps the places of."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as P
from tests import tree_reference as R
from tests.test_gpu_paged_attn_tree import KINDS, Case

pytestmark = pytest.mark.gpu

ROWS = [1, 8, 16, 30, 60, 150]  # times four query heads per KV head: 4 to 600 columns


def _in_a_wide_table(c, blocks):
    """The same sequences in a table with room for many more blocks: their units may be cut."""
    c.table = np.concatenate([c.table, np.full((len(c.table), blocks), -1, np.int32)], 1)
    return c


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n", ROWS)
def test_widths(n, d, pool, dtype):
    c = Case(n + d, [n, 1, n // 2], [700, 90, 40], 8, 2, d, pool, dtype, words=(max(n, 1) + 63) // 64)
    c.check()
    _in_a_wide_table(c, 2000).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 8, 16])
def test_narrow_trees_by_the_tiles_of_all_units(n, d, pool, dtype):
    """Up to 64 columns, cut: parts of a workgroup for fewer than 2048 tiles and from 12288 on, four waves side by side between."""
    c = Case(n + d + 7, [n, 2, n // 2], [900, 77, 30], 8, 2, d, pool, dtype)
    for more in (400, 1500, 6000):
        _in_a_wide_table(c, more).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("n", ROWS)
def test_what_is_not_seen_does_not_matter(n, pool, dtype):
    """NaN in K and V of a new token: only those that see it notice, in any shape of workgroup."""
    c = Case(n, [n], [333], 8, 2, 64, pool, dtype, words=(n + 63) // 64)
    within = c.want(0)
    at = int(c.ctx[0]) - 1 - n // 3
    b = c.table[0, at // c.block], at % c.block
    k, v = c.k16.copy(), c.v16.copy()
    k[b], v[b] = np.nan, np.nan
    c.set_rows(k, v)
    sees = np.asarray(c.seen[0])[:, at - 333]
    for wide in (False, True):
        if wide:
            _in_a_wide_table(c, 2000)
        got = P.from_bits(c.run(), dtype).reshape(within[0].shape)
        assert np.isnan(got[sees]).all()
        P.assert_within(got[~sees], within[0][~sees], within[1][~sees])


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("n", ROWS)
def test_scores_far_apart(n, pool, dtype):
    c = Case(n, [n], [500], 8, 2, 64, pool, dtype, scale=2.0 ** 26, words=(n + 63) // 64)
    rng = np.random.default_rng(n)
    c.q = P.to_bits(rng.integers(-1, 2, c.q.shape), dtype)
    c.set_rows(rng.integers(-1, 2, c.k16.shape).astype(np.float16), c.v16)
    (k, _), (v, _) = c.values(0)
    q, seen = P.from_bits(c.q, dtype).reshape(-1, 8, 64), c.visible(0)
    for wide in (False, True):
        if wide:
            _in_a_wide_table(c, 2000)
        got = P.from_bits(c.run(), dtype).reshape(q.shape)
        for h in range(8):
            score = np.where(seen, q[:, h] @ k[:, h // 4].T, -np.inf)
            w = (score == score.max(1, keepdims=True)).astype(float)
            w /= w.sum(1, keepdims=True)
            want, size = w @ v[:, h // 4], w @ np.abs(v[:, h // 4])
            bound = (2.0 ** -11 + 2.0 ** -16) * size + 2.0 ** -24 * np.abs(v).max() + P.HALF_STEP[dtype] * np.abs(want) + 2.0 ** -25
            P.assert_within(got[:, h], want, bound)


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("d", [32, 64])
def test_few_units_of_many_tiles(d, pool, dtype):
    """One long context, wide enough for four waves: two parts of eight."""
    Case(d, [28], [34000], 32, 8, d, pool, dtype, block=64).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("d,n", [(32, 8), (32, 16), (32, 30), (64, 60), (128, 8)])
def test_more_tiles_than_places(d, n, pool, dtype):
    """Sequences that share their blocks (a common prefix), so many that a workgroup walks through several hundred tiles."""
    hkv, ctx = 8, 17000 if d > 32 else 30000
    c = Case(d + n, [n], [ctx], 4 * hkv, hkv, d, pool, dtype, block=48)
    want, bound = c.want(0)
    seqs = 40
    c.table, c.ctx, c.new = np.repeat(c.table, seqs, 0), np.repeat(c.ctx, seqs), np.repeat(c.new, seqs)
    c.q, c.mask, c.cu, c.total = np.tile(c.q, (seqs, 1)), np.tile(c.mask, (seqs, 1)), np.arange(seqs + 1) * n, seqs * n
    out = P.from_bits(c.run(), dtype).reshape(seqs, *want.shape)
    for s in range(seqs):
        P.assert_within(out[s], want, bound, f"sequence {s}")


def test_no_rows_at_all():
    """Sequences without new rows only, and rows that belong to none: nothing is written."""
    c = Case(1, [3, 2], [50, 20], 4, 2, 64)
    c.cu = np.array([5, 5, 5])
    out = c.run()
    assert (out.view(np.uint8) == 0xFF).all()


@pytest.mark.parametrize("context", [-5, 0, 1, 2])
def test_contexts_shorter_than_the_new_rows(context):
    """New rows whose keys would lie in front of the sequence have none; nothing is read outside the tables."""
    c = Case(2, [5], [0], 4, 2, 64)
    c.ctx = np.array([context])
    out = c.run().astype(np.float64).reshape(5, 4, 64)
    keys = max(context, 0)
    k, v = (x[c.table[0, :1]].reshape(-1, 2, 64)[:keys].astype(np.float64) for x in (c.k, c.v))
    seen = np.asarray(c.seen[0])[:, 5 - keys:] if keys else np.zeros((5, 0), bool)
    want, bound = R.tree_attention(c.q.astype(np.float64).reshape(5, 4, 64), k, v, seen, c.scale, "fp16")
    P.assert_within(out, want, bound)


def test_contexts_beyond_the_table_stop_there():
    c = Case(3, [2], [94], 4, 2, 64)
    c.table = c.table[:, :6].copy()  # 96 rows, all there is
    want = c.run()
    c.ctx = np.array([1 << 30])
    assert np.array_equal(c.run(), want)


@pytest.mark.parametrize("n", [1, 12])
def test_captured_calls_with_a_workspace_each(n):
    """Two graphs replayed at the same time on two streams, their workspaces their own."""
    cases = [Case(40 + i, [n] * 3, [9000, 200, 3000], 8, 2, 64, *KINDS[i]) for i in (0, 2)]
    want = [c.run() for c in cases]
    streams, graphs = [hip.Stream() for _ in cases], []
    for c, s in zip(cases, streams):
        g = hip.Graph(s)
        with g:
            c.launch(s)
        graphs.append(g)
    for _ in range(4):
        for c in cases:
            c.bufs["out"].fill(0xFF)
        hip.synchronize()
        for _ in range(3):
            for g in graphs:
                g.launch()
        hip.synchronize()
        for c, w in zip(cases, want):
            assert np.array_equal(c.bufs["out"].to_numpy(c.q.dtype, c.q.shape), w)
