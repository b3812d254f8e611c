"""Operators over packed rows where what carries the result is far smaller than what lies beside it, or
far larger than a type's ordinary values: against 64-bit forms, within the bounds that the documented
roundings add up to."""
import numpy as np
import pytest

from tests import packed_reference as R
from tests import test_gpu_attn_packed as A

pytestmark = pytest.mark.gpu

FAR = [  # lengths, query and KV heads, head width
    ([1, 33, 150], 4, 2, 64), ([70, 200], 4, 2, 256), ([1090], 4, 2, 64), ([1090], 4, 2, 128),
    ([4097, 4200], 24, 8, 128)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,hq,hkv,d", FAR)
def test_scores_that_are_finite_before_the_scale_only(lens, hq, hkv, d, dtype, causal):
    """All scores of a sequence times the scale lie below what fp32 holds, and their differences are finite (and huge):
    a row is the mean of v over its best keys."""
    one, low, scale = (2.0 ** 8, 2.0 ** 8, 2.0 ** 114) if dtype == "fp16" else (2.0 ** 63, 2.0 ** 62, 16.0)
    rng = np.random.default_rng(3)
    T, n_all = sum(lens) + A.GUARD, sum(lens)
    q, k = np.zeros((T, hq, d)), np.zeros((T, hkv, d))
    q[..., 0] = one
    level = rng.integers(1, 4, T)
    k[..., 0] = -low * level[:, None]  # (times `one` and the scale: at most -2^129)
    v = rng.integers(-8, 9, (T, hkv, d)).astype(np.float64)
    rows = np.concatenate([x.reshape(T, -1) for x in (q, k, v)], 1)
    c = dict(rows=R.to_bits(rows, dtype), lens=lens, hq=hq, hkv=hkv, d=d, dtype=dtype, fused=False, T=T)
    assert (R.from_bits(c["rows"], dtype) == rows).all()
    r = A.Run(c, causal, scale)
    r.launch()
    got = r.result().reshape(n_all, hq, d)
    at = 0
    for n in lens:
        here = level[at:at + n]
        best = np.minimum.accumulate(here) if causal else np.full(n, here.min())
        for h in range(hq):
            vh = v[at:at + n, h // (hq // hkv)]
            want = np.zeros((n, d))
            for b in (1, 2, 3):
                mine = here == b
                if causal:
                    mean = np.cumsum(vh * mine[:, None], 0) / np.maximum(np.cumsum(mine), 1)[:, None]
                else:
                    mean = np.broadcast_to((vh * mine[:, None]).sum(0) / max(mine.sum(), 1), (n, d))
                want[best == b] = mean[best == b]
            # the result's rounding, the reciprocal's and the product's in fp32; sums of ones and integers are exact
            u = R.HALF_STEP[dtype]
            R.assert_within(got[at:at + n, h], want, (u * (1 + 2.0 ** -20) + 3 * R.FP32) * np.abs(want)
                            + (2.0 ** -25 if dtype == "fp16" else 0.0), f"sequence of {n}, head {h}")
        at += n
