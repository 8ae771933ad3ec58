"""Attention operators without a GPU: the oracle's gradients against
differences, the borders of the buckets, and the refusals of the public
functions (every check runs before the device is touched)."""

import numpy as np
import pytest
import torch

from oracle import attention as OA
from rvc_cuda import attention as A


def test_oracle_gradients_against_differences():
    rs = np.random.RandomState(0)
    B, Lq, Lk, Hq, Hkv, D, N = 2, 5, 7, 4, 2, 6, 8
    q, k, v = rs.standard_normal((B, Lq, Hq, D)), rs.standard_normal((B, Lk, Hkv, D)), rs.standard_normal((B, Lk, Hkv, D))
    t, do = rs.standard_normal((N, Hq)), rs.standard_normal((B, Lq, Hq, D))
    live = OA.alive(B, Lq, Lk, kv_lens=[7, 4], causal=True, q_offset=1)
    where = OA.bucket(np.arange(Lk)[None] - np.arange(Lq)[:, None] - 1, N, 6, False)

    def loss(q, k, v, t):
        return (OA.attention(q, k, v, 0.4, live, t.T[:, where])[0] * do).sum()

    got = OA.attention_backward(do, q, k, v, 0.4, live, t.T[:, where], where, N)[:4]
    for n, x in enumerate((q, k, v, t)):
        for at in [tuple(rs.randint(0, s) for s in x.shape) for _ in range(12)]:
            e = np.zeros_like(x)
            e[at] = 1e-5
            args = [q, k, v, t]
            hi, lo = list(args), list(args)
            hi[n], lo[n] = x + e, x - e
            # second-order differences: error about 1e-10 of unit-scale sums
            assert abs((loss(*hi) - loss(*lo)) / 2e-5 - got[n][at]) < 1e-7, (n, at)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_norm_rope_gradient_against_differences(interleaved):
    rs = np.random.RandomState(1)
    x, w, dy = rs.standard_normal((2, 3, 2, 8)), rs.standard_normal(8), rs.standard_normal((2, 3, 2, 8))
    ang = rs.standard_normal((9, 3))
    pos = rs.randint(0, 9, (2, 3))
    f = lambda x, w: (OA.norm_rope(x, w, np.cos(ang), np.sin(ang), pos, 1e-6, interleaved) * dy).sum()  # noqa: E731
    dx, dw = OA.norm_rope_backward(dy, x, w, np.cos(ang), np.sin(ang), pos, 1e-6, interleaved)
    for _ in range(20):
        at = tuple(rs.randint(0, s) for s in x.shape)
        e = np.zeros_like(x)
        e[at] = 1e-5
        assert abs((f(x + e, w) - f(x - e, w)) / 2e-5 - dx[at]) < 1e-7
        e = np.zeros(8)
        e[at[-1]] = 1e-5
        assert abs((f(x, w + e) - f(x, w - e)) / 2e-5 - dw[at[-1]]) < 1e-7


@pytest.mark.parametrize("n,far,both", [(32, 128, True), (32, 128, False), (320, 800, True), (64, 256, True),
                                        (4, 3, True), (2, 5, False), (3, 7, False), (1024, 100000, True),
                                        (6, 1000, False)])
def test_borders_are_the_buckets(n, far, both):
    borders = np.array(A.bucket_borders(n, far, both))
    half = n // 2 if both else n
    assert len(borders) == half - 1 and (np.diff(borders) >= 0).all() and borders[0] >= 1
    r = np.concatenate([np.arange(-3000, 3001), [-far, far, -far - 1, far + 1, -far + 1, far - 1, -10**7, 10**7]])
    a = np.abs(r) if both else np.maximum(-r, 0)
    got = np.searchsorted(borders, a, side="right") + (half * (r > 0) if both else 0)
    np.testing.assert_array_equal(got, OA.bucket(r, n, far, both))


def test_borders_that_fall_on_whole_numbers():
    # e = 8, 8 far buckets, 8 * 16^(k/8) = 8 * 2^(k/2): 16, 32 and 64 open buckets 10, 12 and 14
    b = A.bucket_borders(32, 128, True)
    assert b[:8] == (1, 2, 3, 4, 5, 6, 7, 8) and b[9] == 16 and b[11] == 32 and b[13] == 64


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def refused(match, fn, *a, **k):
    with pytest.raises(ValueError, match=match):
        fn(*a, **k)


def test_attention_refusals():
    q, k = t(2, 5, 4, 16), t(2, 7, 2, 16)
    refused("CUDA", A.attention, q, k, k)
    refused("a tensor", A.attention, q.numpy(), k, k)
    refused("dimensions", A.attention, q[0], k, k)
    refused("float32, bfloat16 or float16", A.attention, q.double(), k, k)
    refused("k: torch.float32", A.attention, q, k.half(), k)
    refused("do not match", A.attention, q, k, t(2, 8, 2, 16))
    refused("do not match", A.attention, q, t(1, 7, 2, 16), t(1, 7, 2, 16))
    refused("do not match", A.attention, q, t(2, 7, 2, 8), t(2, 7, 2, 8))
    refused("no multiple", A.attention, q, t(2, 7, 3, 16), t(2, 7, 3, 16))
    refused("head dimension 129", A.attention, t(1, 1, 1, 129), t(1, 1, 1, 129), t(1, 1, 1, 129))
    refused("kv_lens", A.attention, q, k, k, kv_lens=[1, 2])
    refused("kv_lens", A.attention, q, k, k, kv_lens=t(2))
    refused("kv_lens", A.attention, q, k, k, kv_lens=t(3, dtype=torch.int32))
    refused("key_mask", A.attention, q, k, k, key_mask=t(2, 7))
    refused("key_mask", A.attention, q, k, k, key_mask=t(2, 6, dtype=torch.bool))
    refused("BucketBias", A.attention, q, k, k, bias=t(8, 4))
    refused("q_offset", A._offset, 1.5)
    refused("q_offset", A._offset, (1 << 31) + 1)
    refused("q_offset", A._offset, -(1 << 40))
    refused("4 query heads", A.attention, q, k, k, bias=A.BucketBias(t(8, 2)))
    refused("bias table", A.attention, q, k, k, bias=A.BucketBias(t(8, 4, dtype=torch.float16)))


def test_attention_backward_refusals():
    q, k, lse = t(2, 5, 4, 16), t(2, 7, 2, 16), t(2, 4, 5)
    refused("CUDA", A.attention_backward, q, q, k, k, q, lse)
    refused("dout", A.attention_backward, q[:, :4], q, k, k, q, lse)
    refused("dout", A.attention_backward, q.half(), q, k, k, q, lse)
    refused("out", A.attention_backward, q, q, k, k, q.half(), lse)
    refused("lse", A.attention_backward, q, q, k, k, q, t(2, 5, 4))
    refused("lse", A.attention_backward, q, q, k, k, q, lse.double())


def test_bias_refusals():
    refused("shared by two", A.BucketBias, t(7, 4))
    refused("buckets", A.BucketBias, t(2, 4))
    refused("buckets", A.BucketBias, t(1026, 4))
    refused("max_distance", A.BucketBias, t(32, 4), max_distance=8)
    refused("max_distance", A.BucketBias, t(32, 4), max_distance=1 << 30)
    refused("num_buckets, heads", A.BucketBias, t(32))
    b = A.BucketBias(t(32, 4))
    refused("BucketBias", A.relative_bias, t(32, 4), 3, 3)
    refused("lengths", A.relative_bias, b, -1, 3)
    refused("CUDA", A.relative_bias, b, 3, 3)
    refused("heads", A.relative_bias_backward, b, t(2, 3, 5, 6))
    refused("dbias", A.relative_bias_backward, b, t(2, 4, 5, 6, dtype=torch.float16))
    refused("dimensions", A.relative_bias_backward, b, t(5, 6))
    refused("CUDA", A.relative_bias_backward, b, t(4, 5, 6))


def test_norm_rope_refusals():
    q, k, w, c = t(2, 5, 4, 16), t(2, 5, 2, 16), t(16), t(9, 8)
    f = A.qk_norm_rope
    refused("CUDA", f, q, k, w, w, c, c)
    refused("do not match", f, q, k[:, :4], w, w, c, c)
    refused("head dimension", f, t(1, 1, 1, 15), t(1, 1, 1, 15), t(15), t(15), t(9, 7), t(9, 7))
    refused("head dimension", f, t(1, 1, 1, 258), t(1, 1, 1, 258), t(258), t(258), c, c)
    refused("q_weight", f, q, k, t(8), w, c, c)
    refused("weights", f, q, k, w.half(), w.half(), c, c)
    refused("weights", f, q.half(), k.half(), w.half(), w, c, c)
    refused("cos", f, q, k, w, w, c.half(), c)
    refused("do not fit|fit head", f, q, k, w, w, t(9, 9), t(9, 9))
    refused("fit head", f, q, k, w, w, t(9, 7), c)
    refused("fewer", f, q, k, w, w, t(4, 8), t(4, 8))
    refused("positions", f, q, k, w, w, c, c, positions=t(2, 5))
    refused("positions", f, q, k, w, w, c, c, positions=t(2, 4, dtype=torch.int64))
    refused("dqo", A.qk_norm_rope_backward, q[:, :4], k, q, k, w, w, c, c)
    refused("rope_table", A.rope_table, 4, 7, device="cpu")


def test_rope_table_keeps_far_positions():
    cos, sin = A.rope_table(70000, 16, device="cpu")
    a = 69999 * 10000.0 ** (-np.arange(0, 16, 2) / 16)
    # one rounding to fp32 of values up to 1
    assert np.abs(cos[69999].numpy() - np.cos(a)).max() <= 2.0 ** -24
    assert np.abs(sin[69999].numpy() - np.sin(a)).max() <= 2.0 ** -24


def test_a_table_that_was_replaced():
    """The object's table may be swapped, for one of as many rows only."""
    b = A.BucketBias(t(32, 4))
    for rows in (31, 8, 33, 0):
        b.table = t(rows, 4)
        refused("32 buckets", A.relative_bias, b, 3, 3)
        refused("32 buckets", A.relative_bias_backward, b, t(4, 5, 6))
        refused("32 buckets", A.attention, t(2, 5, 4, 16), t(2, 7, 2, 16), t(2, 7, 2, 16), bias=b)
    b.table = t(32, 4)
    refused("CUDA", A.relative_bias, b, 3, 3)


def test_no_gradient_is_lost_silently():
    """An input that requires grad is refused while grad mode is on; without it the call goes on (to the device)."""
    q, k, w, c, lse = t(2, 5, 4, 16), t(2, 5, 4, 16), t(16), t(9, 8), t(2, 4, 5)
    b, d = A.BucketBias(t(8, 4)), t(4, 5, 5)
    calls = [
        ([q, k, k + 0], lambda q, k, v: A.attention(q, k, v)),
        ([b.table], lambda x: A.attention(q, k, k, bias=A.BucketBias(x))),
        ([q, q + 0, k, k + 0, q + 0, lse], lambda do, q, k, v, o, z: A.attention_backward(do, q, k, v, o, z)),
        ([b.table], lambda x: A.attention_backward(q, q, k, k, q, lse, bias=A.BucketBias(x))),
        ([b.table], lambda x: A.relative_bias(A.BucketBias(x), 3, 3)),
        ([d], lambda x: A.relative_bias_backward(b, x)),
        ([q, k, w, w + 0, c, c + 0], lambda *x: A.qk_norm_rope(*x)),
        ([q, k, w, w + 0, c, c + 0], lambda *x: A.qk_norm_rope(*x, positions=t(2, 5, dtype=torch.int64))),
        ([q, k, q + 0, k + 0, w, w + 0, c, c + 0], lambda *x: A.qk_norm_rope_backward(*x)),
    ]
    for args, fn in calls:
        for n in range(len(args)):
            x = [a.detach().requires_grad_(i == n) for i, a in enumerate(args)]
            refused("requires grad", fn, *x)
            with torch.no_grad():
                refused("CUDA", fn, *x)
    x = torch.nn.Parameter(t(2, 5, 4, 16, 2))[..., 0]  # a view that has to be copied is part of a graph too
    refused("requires grad", A.attention, x, k, k)


def test_a_scale_that_float32_cannot_hold():
    for s in (float("inf"), float("-inf"), float("nan"), 1e39, -1e39, 2.0 ** 127 * (1 + 2.0 ** -50)):
        refused("scale", A._scale, s, 64)
    assert A._scale(2.0 ** 127, 64) == 2.0 ** 127 and A._scale(None, 64) == 0.125


def test_lengths_that_are_no_whole_numbers():
    b = A.BucketBias(t(32, 4))
    for n in (2.5, 3.0, "3", None, -1):
        refused("lengths", A.relative_bias, b, n, 3)
        refused("lengths", A.relative_bias, b, 3, n)
    refused("CUDA", A.relative_bias, b, np.int64(3), 3)


# ------------------------------------------------------- host forms, no torch

WITHOUT_TORCH = """
import sys
sys.path[:0] = {paths!r}
sys.modules["torch"] = None  # an import of torch raises
import numpy as np
from rvc_cuda import ops
"""


def without_torch(body):
    """Runs ``body`` in an interpreter that cannot import torch."""
    import subprocess
    import sys

    from tests.conftest import PKG, ROOT

    r = subprocess.run([sys.executable, "-c", WITHOUT_TORCH.format(paths=[ROOT, PKG]) + body], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_host_forms_refuse_without_torch():
    """The operator module and its refusals (before the device is touched) work where there is no torch."""
    without_torch("""
def refused(word, fn, *a, **k):
    try:
        fn(*a, **k)
    except ValueError as e:
        assert word in str(e), (word, str(e))
    else:
        raise AssertionError(word)

t = lambda *s: np.zeros(s, np.float32)
q, k, w, c, b = t(2, 5, 4, 16), t(2, 7, 2, 16), t(16), t(9, 8), ops.BucketBias(t(8, 4))
refused("dimensions", ops.attention, q[0], k, k)
refused("do not match", ops.attention, q, k, t(2, 8, 2, 16))
refused("no multiple", ops.attention, q, t(2, 7, 3, 16), t(2, 7, 3, 16))
refused("head dimension", ops.attention, t(1, 1, 1, 129), t(1, 1, 1, 129), t(1, 1, 1, 129))
refused("integers", ops.attention, q, k, k, kv_lens=[1.5, 2.0])
refused("kv_lens", ops.attention, q, k, k, kv_lens=[1, 2, 3])
refused("key_mask", ops.attention, q, k, k, key_mask=np.ones((2, 6)))
refused("BucketBias", ops.attention, q, k, k, bias=t(8, 4))
refused("4 query heads", ops.attention, q, k, k, bias=ops.BucketBias(t(8, 2)))
refused("scale", ops.attention, q, k, k, scale=1e39)
refused("q_offset", ops.attention, q, k, k, q_offset=1.5)
refused("shape of q", ops.attention_backward, q[:, :4], q, k, k, q, t(2, 4, 5))
refused("lse", ops.attention_backward, q, q, k, k, q, t(2, 5, 4))
refused("lengths", ops.relative_bias, b, -1, 3)
refused("heads", ops.relative_bias_backward, b, t(3, 5, 6))
refused("dbias", ops.relative_bias_backward, b, t(5, 6))
b.table = t(7, 4)
refused("8 buckets", ops.relative_bias, b, 3, 3)
refused("do not match", ops.qk_norm_rope, q, k, w, w, c, c)
refused("weights", ops.qk_norm_rope, q, q, t(8), w, c, c)
refused("fit head", ops.qk_norm_rope, q, q, w, w, t(9, 9), t(9, 9))
refused("fewer", ops.qk_norm_rope, q, q, w, w, t(4, 8), t(4, 8))
refused("positions", ops.qk_norm_rope, q, q, w, w, c, c, positions=np.zeros((2, 4), int))
refused("gradient", ops.qk_norm_rope_backward, q[:, :4], q, q, q, w, w, c, c)
""")
