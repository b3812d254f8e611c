"""Tree attention where numbers are far from ordinary: scales, scores, exponents of the cache, rows that a token does not see."""
import time

import numpy as np
import pytest

from logismos_amd import hip
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
