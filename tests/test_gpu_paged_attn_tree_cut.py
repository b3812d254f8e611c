"""Tree attention where units are dealt out in shares: more sequences than a wave looks at in one go, heads of 96 in every shape."""
import numpy as np
import pytest

from tests.test_gpu_paged_attn_tree import KINDS, Case

pytestmark = pytest.mark.gpu


def _in_a_wide_table(c, blocks):
    c.table = np.concatenate([c.table, np.full((len(c.table), blocks), -1, np.int32)], 1)
    return c


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (3, 1, 96), (16, 4, 64), (8, 1, 128), (16, 4, 32), (4, 4, 160)])
@pytest.mark.parametrize("seqs", [65, 200])
def test_long_contexts_among_many_sequences(seqs, hq, hkv, d, pool, dtype):
    """Units that are cut lie in the first 64 sequences and behind them; with few KV heads the second launch goes by units, with
    several by cuts."""
    rng = np.random.default_rng(seqs + d)
    new = rng.integers(0, 4, seqs)
    prior = rng.integers(0, 150, seqs)
    for s, (n, p) in {2: (9, 3000), 63: (2, 5001), 64: (17, 2600), 100: (0, 3000), 127: (1, 4000), 128: (5, 7000), 149: (12, 900),
                      199: (3, 6100)}.items():
        if s < seqs:
            new[s], prior[s] = n, p
    c = Case(seqs + hq, new.tolist(), prior.tolist(), hq, hkv, d, pool, dtype, front=2, behind=3)
    c.check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("n", [1, 8, 16, 30, 60, 150])
def test_heads_of_96_by_the_width_of_the_tree(n, pool, dtype):
    c = Case(n, [n, 1, n // 2], [700, 90, 40], 8, 2, 96, pool, dtype, words=(n + 63) // 64)
    c.check()
    for more in (400, 1500, 6000):
        _in_a_wide_table(c, more).check()


@pytest.mark.parametrize("pool,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,n", [(32, 8, 28), (16, 16, 100), (16, 16, 200)])
def test_heads_of_96_over_long_contexts(hq, hkv, n, pool, dtype):
    """Two parts of four waves, and four waves side by side with more columns than they have at a time."""
    Case(n, [n], [34000 if n < 50 else 9000], hq, hkv, 96, pool, dtype, block=64, words=4).check()
