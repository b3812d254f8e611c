"""Operators over packed rows: thousands of sequences (the search for a workgroup's sequence takes several
rounds), up to 63 long ones in the order of their lengths, and every number of K parts of the adapters' first product."""
import numpy as np
import pytest

from tests import test_gpu_adapter_add as D
from tests import test_gpu_attn_packed as A

pytestmark = pytest.mark.gpu


def _lengths(n, seed):
    """Sequences of 0 to 3 rows, with runs of empty ones at the borders of the search's segments and an end that
    belongs to a short segment."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 4, n) if n < 10000 else (rng.random(n) < 0.01) * rng.integers(1, 4, n)
    step = -(-n // 64)
    for border in (step, 2 * step, 40 * step, (n - 1) // step * step):
        lens[max(0, border - 2):border + 2] = 0
    lens[step * 3 - 1:step * 3 + 1] = 3
    lens[-1] = 2
    return [int(x) for x in lens]


@pytest.mark.parametrize("n", [63, 64, 65, 4032, 4033, 4100, 5000, 262145])
def test_attention_of_many_sequences(n):
    lens = _lengths(n, n)
    A._check(A._case(40, lens, 2, 1, 64, "bf16"), True)
    A._check(A._case(41, lens, 3, 3, 32, "fp16"), False)


@pytest.mark.parametrize("n", [63, 64, 65, 4032, 4033, 4100, 5000, 262145])
@pytest.mark.parametrize("max_rank", [16, 72])
def test_adapters_of_many_sequences(n, max_rank):
    lens = _lengths(n, n + 1)
    pick = np.random.default_rng(n).integers(-1, 3, n)
    D._check(D._case(42, lens, pick, [max_rank, 5, 11], max_rank, 72, 64, "bf16"))


def _ordered(n, kind):
    rng = np.random.default_rng(n)
    if kind == "equal":
        return [530] * n
    lens = rng.integers(0, 1200, n)
    lens[::5] = 700  # ties
    lens[1] = 0
    lens[n // 2] += max(0, 513 * n + 1 - lens.sum())
    return [int(x) for x in lens]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["equal", "random"])
@pytest.mark.parametrize("n", [2, 8, 9, 15, 16, 17, 40, 63])
def test_attention_in_the_order_of_lengths(n, kind, causal):
    lens = _ordered(n, kind)
    c = A._case(43, lens, 2, 1, 64, "fp16")
    assert c["T"] > 512 * n  # (what the order is for)
    A._check(c, causal)


def _parts(num_seqs, tokens, max_rank, k):
    """K parts of a launch on 256 compute units, restated."""
    long_seqs = tokens >= 32 * num_seqs
    rt = 1 if not long_seqs or max_rank <= 16 else 2 if max_rank <= 32 else 4
    groups = (tokens // (64 if long_seqs else 16) + num_seqs) * -(-max_rank // (16 * rt))
    steps, parts = -(-k // 32), 1
    while parts < 8 and groups * parts < 512 and steps >= 16 * parts:
        parts *= 2
    rounds = 16 if long_seqs else 32
    whole = -(-(-(-steps // parts)) // rounds) * rounds
    return min(parts, -(-steps // whole))


@pytest.mark.parametrize("dtype,out", D.OUTS)
@pytest.mark.parametrize("lens,max_rank,k,parts", [
    ([1, 3, 1], 128, 8192, 8), ([1, 3, 1], 128, 6656, 7), ([1, 3, 1], 128, 6136, 6), ([1, 3, 1], 128, 5000, 5),
    ([70, 33], 72, 4096, 8), ([70, 33], 72, 3328, 7), ([70, 33], 72, 2888, 6), ([70, 33], 16, 4096, 8),
    ([70, 33], 32, 2888, 6), ([1050, 1050], 256, 2048, 4), ([1050, 1050], 256, 1536, 3)], ids=lambda v: str(v))
def test_parts_of_the_first_product(lens, max_rank, k, parts, dtype, out):
    c = D._case(44, lens, np.arange(len(lens)) % 2, [max_rank, max_rank - 3], max_rank, 136, k, dtype, out)
    assert _parts(len(lens), c["T"], max_rank, k) == parts
    D._check(c)
