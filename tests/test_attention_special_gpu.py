"""Attention operators where values are not ordinary: finite results are held
against the 64-bit oracle with the bounds of ``test_attention_gpu`` (its
``Case``), the others are told by their kind alone.
"""

import pytest
import torch

from tests.test_attention_gpu import Case

pytestmark = pytest.mark.gpu

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
