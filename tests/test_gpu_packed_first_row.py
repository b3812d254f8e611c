"""Operators over packed rows whose first sequence starts behind the first row: the rows in front of it are neither
read nor written."""
import numpy as np
import pytest

from logismos_amd import hip
from tests import packed_reference as R
from tests import test_gpu_adapter_add as D
from tests import test_gpu_attn_packed as A

pytestmark = pytest.mark.gpu

FRONT = [1, 15, 16, 17, 64, 130, 700]
LENS = [[1], [5, 0, 33], [200, 1, 64], [1] * 70, [1500]]


def _cu(front, lens):
    return hip.DeviceBuffer.from_numpy((front + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32))


@pytest.mark.parametrize("front", FRONT)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)} of {max(v)}")
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (6, 2, 128)])
def test_attention(hq, hkv, d, lens, front):
    c = A._case(60, [front] + lens, hq, hkv, d, "bf16")
    q, k, v = (x.copy() for x in A._parts(c))
    want, bound = A._want(c, True)
    for x in (q, k, v):
        x[:front] = A._nan("bf16")
    c["rows"], c["lens"] = np.concatenate([q, k, v], 1), lens
    r = A.Run(c, True)
    r.cu = _cu(front, lens)
    r.launch()
    got = r.bits()
    n = front + sum(lens)
    assert (got[:front] == 0xFFFF).all() and (got[n:] == 0xFFFF).all()
    R.assert_within(R.from_bits(got[front:n], "bf16"), want[front:], bound[front:])


@pytest.mark.parametrize("front", FRONT)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)} of {max(v)}")
@pytest.mark.parametrize("max_rank", [16, 64, 72])
@pytest.mark.parametrize("in_place", [False, True])
def test_adapters(in_place, max_rank, lens, front):
    pick = np.arange(len(lens)) % 3 - (len(lens) > 1)
    c = D._case(61, [front] + lens, np.concatenate([[-1], pick]), [max_rank, 5, max_rank - 3], max_rank, 136, 264,
                "bf16")
    want, bound = D._want(c)
    c["x"][:front] = D.NAN["bf16"]
    c["lens"], c["pick"] = lens, pick.astype(np.int32)
    r = D.Run(c, in_place)
    r.cu = _cu(front, lens)
    r.launch()
    got, n = r.bits(), front + sum(lens)
    for rows in (slice(0, front), slice(n, None)):
        assert np.array_equal(got[rows], c["base"][rows]) if in_place else (got[rows] == 0xFFFF).all()
    R.assert_within(R.from_bits(got[front:n], "bf16"), want[front:], bound[front:])
