"""The adapters' workspace: no larger than the parts of the first product that a launch can make, and enough
for every batch that is smaller than the one it was asked for."""
import numpy as np
import pytest

from logismos_amd import hip, kernels
from tests import packed_reference as R
from tests import test_gpu_adapter_add as D

size = kernels.adapter_add_workspace_bytes


def _parts(num_seqs, tokens, max_rank, k, units):
    """K parts of a launch, restated."""
    long_seqs = tokens >= 32 * num_seqs
    rt = 1 if not long_seqs or max_rank <= 16 else 2 if max_rank <= 32 else 4
    groups = (tokens // (64 if long_seqs else 16) + num_seqs) * -(-max_rank // (16 * rt))
    steps, parts = -(-k // 32), 1
    while parts < 8 and groups * parts < 2 * units and steps >= 16 * parts:
        parts *= 2
    return parts


def test_a_long_prefill_asks_for_one_part():
    assert size(1 << 16, 256) == (1 << 16) * 256 * 4
    assert size(1 << 23, 256) == (1 << 23) * 256 * 4
    assert size(131072, 64) == 131072 * 64 * 4


def test_few_rows_ask_for_all_parts():
    assert size(1, 8) == 8 * 8 * 4 and size(200, 64) == 8 * 200 * 64 * 4


@pytest.mark.parametrize("max_rank", range(8, 264, 8))
def test_it_is_enough(max_rank):
    rng = np.random.default_rng(max_rank)
    edges = [64 * i + j for i in (1, 31, 32, 63, 64, 127, 128, 255, 256, 511, 512) for j in (-1, 0, 1)]
    tokens = edges + [int(np.exp(rng.uniform(0, np.log(1 << 22)))) for _ in range(60)]
    for t in tokens:
        for num_seqs in {1, 2, max(1, t // 32), max(1, t // 33), t, t + 5}:
            for k in (8, 1 << 9, 1 << 13, 1 << 22):
                for units in (32, 256):
                    need = 4 * t * max_rank * _parts(num_seqs, t, max_rank, k, units)
                    assert need <= size(t, max_rank)


def test_it_never_shrinks():
    tokens = sorted({int(2 ** (i / 8)) for i in range(23 * 8 + 1)})
    for r in range(8, 264, 8):
        sizes = [size(t, r) for t in tokens]
        assert sizes == sorted(sizes)
    for t in tokens:
        sizes = [size(t, r) for r in range(8, 264, 8)]
        assert sizes == sorted(sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,max_rank,k", [
    ([4096], 64, 1024), ([8000, 60], 16, 512), ([1024], 256, 2048), ([33] * 200, 128, 1024), ([1] * 2000, 8, 512),
    ([1], 72, 4096), ([16383], 32, 640)], ids=lambda v: str(v)[:20])
def test_nothing_behind_it_is_written(lens, max_rank, k):
    c = D._case(30, lens, np.arange(len(lens)) % 2, [max_rank, max_rank - 3], max_rank, 64, k, "bf16")
    r = D.Run(c)
    n = size(c["T"], max_rank)
    r.ws = hip.DeviceBuffer(n + 65536)
    r.ws.fill(0xFF)
    r.launch()
    got = r.bits()
    assert (r.ws.to_numpy(np.uint8, (n + 65536,))[n:] == 0xFF).all()
    rows = sum(lens)
    R.assert_within(R.from_bits(got[:rows, :64], "bf16"), *D._want(c))
