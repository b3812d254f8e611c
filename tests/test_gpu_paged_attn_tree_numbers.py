"""Tree attention where numbers are far from ordinary: scales, scores, exponents of the cache, rows that a token does not see."""
import numpy as np
import pytest

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
