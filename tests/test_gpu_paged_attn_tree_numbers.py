"""Tree attention where numbers are far from ordinary: scales, scores, exponents of the cache, rows that a token does not see."""
import time

import numpy as np
import pytest

from logismos_amd import hip
from tests import packed_reference as P
from tests import tree_reference as R
from tests.test_gpu_paged_attn_tree import KINDS, Case

pytestmark = pytest.mark.gpu

ROWS = [1, 8, 16, 30, 60]  # times four query heads per KV head


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("scale", [1e-7, 1e-8, 1e-20])
def test_small_scales(scale, n, pool, dtype):
    """Every key weighs the same, also beside tiles that are not there: behind the last one of a part, in holes of the table."""
    c = Case(n, [n, 3], [300, 40], 8, 2, 64, pool, dtype, scale=scale)
    c.check()
    c.table = np.concatenate([c.table, np.full((2, 2000), -1, np.int32)], 1)
    c.check()


def test_rows_that_nobody_sees_take_no_time():
    """What lies behind the last row of a sequence, in a block that is not full: NaN there costs what zeros do."""
    seqs, ctx, n, d = 40, 17001, 8, 64
    c = Case(5, [n], [ctx - n], 32, 8, d, "e4m3", "fp16", block=48)
    c.table, c.ctx, c.new = np.repeat(c.table, seqs, 0), np.repeat(c.ctx, seqs), np.repeat(c.new, seqs)
    c.q, c.mask, c.cu, c.total = np.tile(c.q, (seqs, 1)), np.tile(c.mask, (seqs, 1)), np.arange(seqs + 1) * n, seqs * n
    last, used = c.table[0, (ctx - 1) // 48], ctx % 48
    assert 0 < used < 47
    times, outs = [], []
    for fill in (0, 0x7F):
        for pool in (c.k, c.v):
            pool[last, used:] = fill
        c.upload()
        best = np.inf
        for _ in range(12):
            hip.synchronize()
            t = time.perf_counter()
            for _ in range(5):
                c.launch()
            hip.synchronize()
            best = min(best, time.perf_counter() - t)
        times.append(best)
        outs.append(c.bufs["out"].to_numpy(c.q.dtype, c.q.shape))
    assert np.array_equal(*outs)
    assert times[1] < 1.4 * times[0], times


def _wide(c, blocks=2000):
    """The same sequences in a table with room for many more blocks: their units may be cut."""
    c.table = np.concatenate([c.table, np.full((len(c.table), blocks), -1, np.int32)], 1)
    return c


def _drafted(c, s, j):
    """Block and row of drafted token j of sequence s."""
    at = int(c.ctx[s] - c.new[s]) + j
    return c.table[s, at // c.block], at % c.block


def _bounded_by_what_is_seen(c, s):
    """The formula row by row, the bound of each by the exponents of those keys alone that it sees."""
    (k, ke), (v, ve) = c.values(s)
    seen = c.visible(s)
    q = P.from_bits(c.q[c.cu[s]:c.cu[s + 1], :c.hq * c.d], c.dtype).reshape(-1, c.hq, c.d)
    found = []
    for i in range(len(q)):
        mine = seen[i:i + 1]
        only = [np.where(mine[0][:, None], e, R.LOWEST) for e in (ke, ve)]
        found.append(R.tree_attention(q[i:i + 1], *(np.where(mine[0][:, None, None], x, 0.0) for x in (k, v)), mine, c.scale,
                                      c.dtype, *only))
    return [np.concatenate(x) for x in zip(*found)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("n", ROWS[1:])
def test_large_rows_of_other_branches(n, which, dtype):
    """Finite rows at the cache's largest exponent (and bytes beyond it) that some tokens do not see: to those they might as well be
    zeros, bit for bit; those that see the V row get what the formula gives."""
    for exponent in (32, 14, 128):
        c = Case(n, [n, 3 + n // 2], [333, 64], 8, 2, 64, "e4m3", dtype)
        hit = [(s, int(c.new[s]) // 2) for s in range(2)]
        for s, j in hit:  # (what the others see, with nothing there)
            b, row = _drafted(c, s, j)
            c.k[b, row] = c.v[b, row] = 0
            c.k_exp[b, :, row] = c.v_exp[b, :, row] = 127 + R.LOWEST
        for wide in (False, True):
            if wide:
                _wide(c)
            clean = c.run()
            kept = c.k.copy(), c.v.copy(), c.k_exp.copy(), c.v_exp.copy()
            rng = np.random.default_rng(n)
            for s, j in hit:
                b, row = _drafted(c, s, j)
                for name in "kv" if which == "both" else which:
                    getattr(c, name)[b, row] = rng.integers(0x60, 0x7F, (2, 64)) | rng.integers(0, 2, (2, 64)) * 0x80
                    getattr(c, name + "_exp")[b, :, row] = 127 + exponent
            out = c.run()
            for s, j in hit:
                rows, sees = np.arange(c.cu[s], c.cu[s + 1]), np.asarray(c.seen[s])[:, j]
                assert (~sees).any() and np.array_equal(out[rows[~sees]], clean[rows[~sees]])
                if which == "v" and exponent < 127 and dtype == "bf16":
                    want, bound = _bounded_by_what_is_seen(c, s)
                    P.assert_within(P.from_bits(out[rows], dtype).reshape(want.shape), want, bound, f"sequence {s}")
            c.k, c.v, c.k_exp, c.v_exp = kept


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n", ROWS)
def test_drafted_rows_of_any_exponents(n, dtype):
    """Drafted K and V rows from 2^-60 to 2^10 of one another; every row to a bound of what it sees itself."""
    c = Case(n + 50, [n, 2 * n // 3 + 1], [90, 0], 8, 2, 64, "e4m3", dtype)
    rng = np.random.default_rng(n)
    for s in range(2):
        for j in range(int(c.new[s])):
            b, row = _drafted(c, s, j)
            c.k_exp[b, :, row] = 127 + rng.integers(-40, -6, 2)
            c.v_exp[b, :, row] = 127 + rng.integers(-64, 5, 2)
    for wide in (False, True):
        if wide:
            _wide(c)
        out = c.run()
        for s in range(2):
            want, bound = _bounded_by_what_is_seen(c, s)
            P.assert_within(P.from_bits(out[c.cu[s]:c.cu[s + 1]], dtype).reshape(want.shape), want, bound, f"sequence {s}")


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("n", [1, 16, 60])
@pytest.mark.parametrize("shift,low", [(120, 0), (126, 0), (126, 300), (90, 0)])
def test_scores_that_are_beyond_fp32_with_the_scale(shift, low, n, pool, dtype):
    """Whole numbers as scores (less `low`, the same for all keys), times a scale with which they are no numbers of 32 bits: the keys
    with the largest share all the weight.  e4m3: also with K at the cache's largest exponent."""
    for exponent in (None, 32) if pool == "e4m3" else (None,):
        c = Case(n + shift, [n, 3], [300, 40], 8, 2, 64, pool, dtype, scale=2.0 ** shift)
        rng = np.random.default_rng(n)
        q, k = rng.integers(-1, 2, c.q.shape), rng.integers(-1, 2, c.k16.shape)
        q.reshape(-1, 8, 64)[..., 0], k[..., 0] = 16, -low / 16
        c.q = P.to_bits(q, dtype)
        if pool == "e4m3":
            k[..., 0] = -low // 16 // 2 * 2  # (a number of e4m3 beside 1)
        c.set_rows(k.astype(np.float16), c.v16)
        if exponent is not None:
            c.k_exp[:] = 127 + exponent
        for wide in (False, True):
            if wide:
                _wide(c)
            out = c.run()
            for s in range(2):
                (k, _), (v, ve) = c.values(s)
                q = P.from_bits(c.q[c.cu[s]:c.cu[s + 1]], dtype).reshape(-1, 8, 64)
                got, seen = P.from_bits(out[c.cu[s]:c.cu[s + 1]], dtype).reshape(q.shape), c.visible(s)
                for h in range(8):
                    score = np.where(seen, q[:, h] @ k[:, h // 4].T, -np.inf)
                    w = (score == score.max(1, keepdims=True)).astype(float)
                    w /= w.sum(1, keepdims=True)
                    want, size = w @ v[:, h // 4], w @ np.abs(v[:, h // 4])
                    # equal weights, off by half a step of fp16 and by fp32 sums; of neighbours' rows of V 2^-25 of the largest step
                    bound = (2.0 ** -11 + 2.0 ** -16) * size + 2.0 ** -24 * np.abs(v).max() + P.HALF_STEP[dtype] * np.abs(want) + 2.0 ** -25
                    P.assert_within(got[:, h], want, bound)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("scale", [1e-30, 1e-37])
def test_scales_that_vanish_beside_the_exponents_of_k(scale, dtype):
    """Rows of K at the cache's lowest exponent: every key weighs the same."""
    c = Case(3, [20, 5], [200, 31], 8, 2, 64, "e4m3", dtype, scale=scale)
    c.k_exp[:] = 127 - 64
    c.check()
    _wide(c).check()
