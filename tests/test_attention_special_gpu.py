"""Attention operators where values are not ordinary: finite results are held
against the 64-bit oracle with the bounds of ``test_attention_gpu`` (its
``Case``), the others are told by their kind alone.
"""

import numpy as np
import pytest
import torch

from tests.test_attention_gpu import Case, f8

pytestmark = pytest.mark.gpu

from rvc_cuda import attention as A  # noqa: E402

# B, Hq, Hkv, D, Lq, Lk: few rows (one launch, a cluster, the workspace), the general kernels with one and
# several splits, the tiles of 16 bits, those of fp32
PATHS = [
    (2, 2, 2, 64, 1, 40), (2, 12, 12, 64, 1, 499), (1, 4, 2, 128, 3, 4100), (2, 4, 2, 33, 20, 70), (1, 6, 3, 24, 18, 2100),
    (2, 2, 1, 64, 130, 700), (1, 4, 2, 128, 70, 2100), (2, 2, 2, 96, 100, 400), (1, 2, 1, 40, 300, 300),
]


# ------------------------------------------------------- behind a causal limit


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", PATHS, ids=str)
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_keys_past_the_causal_limit_hold_anything(dtype, size, junk):
    """A preallocated cache: what lies past the last query's limit is not written yet."""
    B, Lq, Lk = size[0], size[4], size[5]
    for off, kw in ((2, {}), (Lk // 3 - Lq, dict(lens=[Lk] + [Lk // 2] * (B - 1))), (Lk - Lq - 1, {}),
                    (-Lq // 2, dict(keep="random") if B > 1 else {})):
        c = Case(dtype, *size, causal=True, q_offset=off, **kw)
        dead = torch.from_numpy(~c.live.any(1)).cuda()[:, :, None, None]
        c.k, c.v = c.k.masked_fill(dead, junk), c.v.masked_fill(dead, junk)
        c.forward()
        c.backward()


# ------------------------------------------------------ live NaN and infinities


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", PATHS, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_live_values_that_are_not_finite_are_seen(dtype, size, bad):
    """They come out as NaN in the rows that meet them, in the log sum too, and
    nowhere else; 0 and -inf are left to queries without a live key."""
    B, Hq, Hkv, D, Lq, Lk = size
    g = Hq // Hkv
    for key in (0, Lk // 2, Lk - 1):
        c = Case(dtype, *size)
        i, h = Lq // 2, Hkv - 1
        q = c.q.clone()
        q[B - 1, i, h * g] = bad  # a query: every score of its row
        out, lse = A.attention(q, c.k, c.v)
        hit = np.zeros((B, Lq, Hq), bool)
        hit[B - 1, i, h * g] = True
        assert np.isnan(f8(out)[hit]).all() and np.isnan(f8(lse).transpose(0, 2, 1)[hit]).all(), "query"
        assert np.isfinite(f8(out)[~hit]).all() and np.isfinite(f8(lse).transpose(0, 2, 1)[~hit]).all(), "other queries"
        k = c.k.clone()
        k[B - 1, key, h] = bad  # a key: NaN, or an infinite score in every row of its heads
        out, lse = A.attention(torch.ones_like(c.q) * (1 if bad > 0 else -1), k, c.v)
        hit = np.zeros((B, Lq, Hq), bool)
        hit[B - 1, :, h * g:(h + 1) * g] = True
        assert np.isnan(f8(out)[hit]).all() and np.isnan(f8(lse).transpose(0, 2, 1)[hit]).all(), "key"
        assert np.isfinite(f8(out)[~hit]).all() and np.isfinite(f8(lse).transpose(0, 2, 1)[~hit]).all(), "other heads"
        v = c.v.clone()
        v[B - 1, key, h, D - 1] = bad  # a value: its column of the outputs, no log sum
        out, lse = A.attention(c.q, c.k, v)
        col = np.zeros((B, Lq, Hq, D), bool)
        col[B - 1, :, h * g:(h + 1) * g, D - 1] = True
        assert not np.isfinite(f8(out)[col]).any() and np.isfinite(f8(out)[~col]).all() and np.isfinite(f8(lse)).all(), "value"
