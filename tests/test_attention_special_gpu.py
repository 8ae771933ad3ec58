"""Attention operators where values are not ordinary: finite results are held
against the 64-bit oracle with the bounds of ``test_attention_gpu`` (its
``Case``), the others are told by their kind alone.
"""

import numpy as np
import pytest
import torch

from oracle import attention as OA
from tests.test_attention_gpu import Case, f8

pytestmark = pytest.mark.gpu

from rvc_cuda import _lib, attention as A  # noqa: E402

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


# ------------------------------------------------- table entries that mask


def with_table(c, rows, value):
    """``c`` with rows of its table set, and what the oracle says of it: an entry
    whose scaled form leaves float32 (-inf, the lowest bfloat16 and float32)
    masks the pairs of its bucket."""
    t = c.kw["bias"].table
    t[rows] = value
    tab = f8(t)
    tab = np.where(tab * np.log2(np.e) < np.finfo(np.float32).min, -np.inf, tab)
    c.tab = tab.T[:, c.where]
    rep = lambda x: np.repeat(x, c.g, 2)  # noqa: E731
    c.out, c.lse, c.p = OA.attention(c.q8, c.k8, c.v8, c.scale, c.live, c.tab)
    s = OA.scores(c.q8, c.k8, c.scale, c.live, c.tab)
    mag = np.einsum("bihd,bjhd->bhij", np.abs(c.q8), rep(np.abs(c.k8))) * abs(c.scale)
    c.es = np.where(np.isfinite(s), 2.0 ** -20 * mag + 2.0 ** -21 * np.abs(np.where(np.isfinite(s), s, 0)), 0.0)
    c.ep = 2 * c.es.max(-1, keepdims=True, initial=0.0) + 2.0 ** -20
    c.pv = np.einsum("bhij,bjhd->bihd", c.p * (c.ep + c.w), rep(np.abs(c.v8)))
    return c


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("value", ["-inf", "lowest"])
@pytest.mark.parametrize("size", [(2, 4, 2, 64, 3, 900), (1, 2, 2, 40, 150, 700), (1, 2, 1, 128, 300, 900),
                                  (1, 2, 2, 64, 70, 4100), (1, 2, 1, 96, 80, 260)], ids=str)
def test_a_masked_bucket(dtype, value, size):
    """A window: the far buckets are masked.  Queries meet far tiles first, some
    meet nothing else; scores are large enough to overflow fp16 weights that
    forget the bias."""
    Lk = size[5]
    for both, off, rows in ((True, Lk // 2, [3, 7]), (True, 5000, [3, 7]), (True, -5000, [7]), (False, Lk // 2, [7]),
                            (True, 40, slice(None))):
        c = Case(dtype, *size, bias=(8, 6, both), q_offset=off, scale=3.0 / np.sqrt(size[3]))
        c = with_table(c, rows, float("-inf") if value == "-inf" else torch.finfo(c.t).min)
        c.forward()
        c.backward()


def test_the_entry_points_refuse_a_scale_that_float32_cannot_hold():
    c = Case("bf16", 1, 1, 1, 64, 1, 40)
    desc = (A.C.c_int64 * 29)(1, 1, 1, 1, 1, 40, 64, *c.q.stride()[:3], *c.k.stride()[:3], *c.v.stride()[:3], 0, 0, 0, 0, 0,
                              0, 0, *c.do.stride()[:3], *c.q.stride()[:3])
    ctx, lse = _lib.get_context().handle, torch.zeros(1, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    o = [torch.empty_like(x) for x in (c.q, c.q, c.k, c.v)]
    p = [x.data_ptr() for x in (c.do, c.q, c.k, c.v, *o, lse, ws)]
    n0 = _lib.launch_count()
    for s in (1e39, float("inf"), float("nan")):
        assert _lib.lib.rvc_cuda_attention_device(ctx, None, desc, 29, s, *p[1:4], None, None, None, None, 0, p[4], p[8], p[9],
                                                  1 << 20) == _lib.RVC_E_ARG
        assert _lib.lib.rvc_cuda_attention_backward_device(ctx, None, desc, 29, s, *p[:5], p[8], None, None, None, None, 0,
                                                           *p[5:8], None, p[9], 1 << 20) == _lib.RVC_E_ARG
        assert "scale" in _lib.last_error()
    assert _lib.launch_count() == n0


# ----------------------------------------------------------- infinite gradients


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", [(1, 2, 1, 64, 1, 40), (2, 2, 2, 33, 5, 70), (1, 2, 1, 64, 80, 300), (1, 1, 1, 128, 9, 400)],
                         ids=str)
def test_an_infinite_gradient_is_seen(dtype, size):
    """A loss scale that overflowed: dq and dk must not look as if nothing was."""
    for bad in (float("inf"), float("-inf"), float("nan")):
        c = Case(dtype, *size)
        i, h, g = size[4] // 2, 0, size[1] // size[2]
        v, do = c.v.abs() + 0.1, c.do.clone()
        do[0, i, h, 1] = bad
        out, lse = A.attention(c.q, c.k, v)
        dq, dk, dv = A.attention_backward(do, c.q, c.k, v, out, lse)
        assert not torch.isfinite(dq[0, i, h]).any() and torch.isfinite(dq[0, i, g:]).all()
        assert not torch.isfinite(dk[0, :, 0]).any() and not torch.isfinite(dv[0, :, 0, 1]).any()
        assert torch.isfinite(dk[1:]).all() and torch.isfinite(dv[1:]).all() and torch.isfinite(dq[1:]).all()


# --------------------------------------------------- queries that meet one key


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", [(2, 4, 2, 64, 70, 300), (2, 2, 1, 128, 150, 400), (2, 3, 3, 40, 9, 700),
                                  (2, 2, 2, 64, 300, 300), (2, 2, 1, 64, 5, 40)], ids=str)
def test_queries_with_one_live_key(dtype, size):
    """A softmax over one key is 1, whether the length, the mask or the causal
    limit leaves it: exactly no gradient reaches q, the key or the table from there."""
    B, Lq, Lk = size[0], size[4], size[5]
    one = np.zeros((B, Lk), bool)
    one[0, 0] = one[1, Lk - 1] = True
    two = one.copy()
    two[:, Lk // 2] = True
    none = one.copy()
    none[1] = False
    one, two, none = one.tolist(), two.tolist(), none.tolist()
    for kw in (dict(lens=[1, 1]), dict(keep=one), dict(keep=none), dict(causal=True), dict(keep=two, causal=True, q_offset=3),
               dict(keep=two, lens=[Lk, Lk // 2 + 1]), dict(causal=True, q_offset=1 - Lq), dict(lens=[1, Lk], causal=True)):
        c = Case(dtype, *size, bias=(8, 6, True), **kw)
        dq, dk, _, dt = c.backward()
        lone = torch.from_numpy(c.live.sum(-1) <= 1).cuda()
        assert (dq[lone] == 0).all(), kw
        for b in range(B):
            assert not lone[b].all() or (dk[b] == 0).all(), kw
        assert not lone.all() or (dt == 0).all(), kw


# ------------------------------------------------- table rows that no pair uses


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", [(1, 2, 2, 64, 70, 300), (2, 4, 2, 128, 129, 260), (1, 2, 1, 40, 5, 270), (1, 2, 1, 64, 3, 50)],
                         ids=str)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_entries_that_no_pair_uses_reach_nothing(dtype, size, value):
    """Buckets past the call's distances may hold anything: rows and keys that pad
    a tile lie at such distances."""
    for both, off in ((True, 0), (True, size[5] - size[4]), (False, size[5]), (True, 2 * size[5])):
        c = Case(dtype, *size, bias=(64, 8000, both), q_offset=off, lens=[size[5]] + [size[5] - 7] * (size[0] - 1))
        used = np.unique(c.where[c.live.any(0)])
        rest = torch.ones(64, dtype=torch.bool, device="cuda")
        rest[torch.from_numpy(used).cuda()] = False
        c.kw["bias"].table[rest] = value
        c.forward()
        got = c.backward()
        assert all(torch.isfinite(x).all() for x in got)


# ------------------------------------------------- table entries far below zero


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("value", [-70000.0, -1e9, -1e30])
@pytest.mark.parametrize("size", [(2, 4, 2, 64, 3, 900), (1, 2, 2, 40, 150, 700), (1, 2, 1, 128, 300, 900), (1, 2, 2, 64, 70, 4100)],
                         ids=str)
def test_entries_far_below_zero_mask(dtype, value, size):
    """Queries whose every pair has such an entry have no live key; the gradients
    of the others are what they are without those pairs."""
    Lk = size[5]
    for both, off, rows in ((True, Lk // 2, [3, 7]), (True, 5000, [3, 7]), (True, -5000, [7]), (False, Lk // 2, [7]),
                            (True, 40, slice(None))):
        c = Case(dtype, *size, bias=(8, 6, both), q_offset=off)
        c = with_table(c, rows, float("-inf"))
        c.kw["bias"].table[rows] = value
        c.forward()
        c.backward()


# ----------------------------------------------------- pointers of the C calls


def test_the_entry_points_refuse_misaligned_lengths_tables_and_positions():
    """A value that lies across its size would fault the device: refused before any launch."""
    c = Case("fp32", 2, 2, 2, 64, 3, 40, lens=[40, 3], bias=(8, 6, True))
    ctx, n0 = _lib.get_context().handle, _lib.launch_count()
    bias, borders, nb = c.kw["bias"], c.kw["bias"]._borders, c.kw["bias"]._nborders
    room = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    at = room.data_ptr()
    o = [torch.empty_like(x) for x in (c.q, c.q, c.k, c.v)]
    p = [x.data_ptr() for x in (c.do, c.q, c.k, c.v, *o)]
    lse = torch.zeros(2, 2, 3, device="cuda").data_ptr()
    for bits, lens, table, word in ((32, at + 2, at, "kv_lens"), (64, at + 4, at, "kv_lens"), (32, at, at + 2, "table")):
        desc = (A.C.c_int64 * 29)(0, 2, 2, 2, 3, 40, 64, *c.q.stride()[:3], *c.k.stride()[:3], *c.v.stride()[:3], bits, 0, 0,
                                  0, 0, 8, 1, *c.do.stride()[:3], *c.q.stride()[:3])
        assert _lib.lib.rvc_cuda_attention_device(ctx, None, desc, 29, 0.125, *p[1:4], lens, None, table, borders, nb, p[4],
                                                  lse, at, 1 << 20) == _lib.RVC_E_ARG
        assert word in _lib.last_error() and "misaligned" in _lib.last_error()
        assert _lib.lib.rvc_cuda_attention_backward_device(ctx, None, desc, 29, 0.125, *p[:4], p[4], lse, lens, None, table,
                                                           borders, nb, *p[5:8], bias.table.data_ptr(), at, 1 << 20) == _lib.RVC_E_ARG
        assert word in _lib.last_error() and "misaligned" in _lib.last_error()
    cos, sin = (x.data_ptr() for x in A.rope_table(9, 64, device="cuda"))
    w = torch.ones(64, device="cuda").data_ptr()
    for bits, pos in ((32, at + 2), (64, at + 4)):
        desc = (A.C.c_int64 * 25)(0, 0, 2, 3, 2, 2, 64, 64, 9, 0, bits, 3, 1, *c.q.stride()[:3], *c.q.stride()[:3],
                                  *c.q.stride()[:3], *c.q.stride()[:3])
        assert _lib.lib.rvc_cuda_qk_norm_rope_device(ctx, None, desc, 25, 1e-6, p[1], p[1], w, w, cos, sin, pos, p[4],
                                                     p[5]) == _lib.RVC_E_ARG
        assert "misaligned positions" in _lib.last_error()
        assert _lib.lib.rvc_cuda_qk_norm_rope_backward_device(ctx, None, desc, 25, 1e-6, p[0], p[0], p[1], p[1], w, w, cos,
                                                              sin, pos, p[4], p[5], w, w, at, 1 << 20) == _lib.RVC_E_ARG
        assert "misaligned positions" in _lib.last_error()
    assert _lib.launch_count() == n0


# ------------------------------------------------------------------ host forms


def test_host_forms_without_torch():
    """The numpy forms run where torch cannot be imported."""
    from tests.test_attention import without_torch

    without_torch("""
from oracle import attention as OA
rs = np.random.RandomState(0)
n = lambda *s: rs.standard_normal(s).astype(np.float32)
q, k, v, do, bias = n(2, 30, 4, 32), n(2, 41, 2, 32), n(2, 41, 2, 32), n(2, 30, 4, 32), ops.BucketBias(n(16, 4), 30, True)
lens = np.array([41, 20])
out, lse = ops.attention(q, k, v, kv_lens=lens, bias=bias)
live = OA.alive(2, 30, 41, lens)
where = OA.bucket(np.arange(41)[None] - np.arange(30)[:, None], 16, 30, True)
o, z, _ = OA.attention(q, k, v, 32 ** -0.5, live, bias.table.T[:, where])
assert np.abs(out - o).max() <= 2.0 ** -15 and np.abs(lse - z).max() <= 2.0 ** -15
got = ops.attention_backward(do, q, k, v, out, lse, kv_lens=lens, bias=bias)
want = OA.attention_backward(do, q, k, v, 32 ** -0.5, live, bias.table.T[:, where], where, 16)
for a, b in zip(got, want):
    assert np.abs(a - b).max() <= 2.0 ** -13 * max(1.0, np.abs(b).max())
assert (ops.relative_bias(bias, 30, 41) == bias.table.T[:, where]).all()
assert ops.relative_bias_backward(bias, n(4, 30, 41)).shape == (16, 4)
g, ang = n(32), n(41, 16)
a, b = ops.qk_norm_rope(k, v, g, g, np.cos(ang), np.sin(ang))
pos = np.broadcast_to(np.arange(41), (2, 41))
assert np.abs(b - OA.norm_rope(v, g, np.cos(ang), np.sin(ang), pos, 1e-6, False)).max() <= 2.0 ** -17 * 16
assert len(ops.qk_norm_rope_backward(a, b, k, v, g, g, np.cos(ang), np.sin(ang), positions=np.arange(41))) == 4
""")


def test_host_forms_are_the_tensor_forms():
    """Same bits as the calls on tensors, empty sizes and every option included."""
    from rvc_cuda import ops

    rs = np.random.RandomState(1)
    n = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731

    def same(a, b):
        a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
        assert len(a) == len(b)
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y.cpu().numpy())

    for B, Lq, Lk, Hq, Hkv, D in ((2, 30, 41, 4, 2, 32), (1, 1, 300, 3, 3, 7), (2, 70, 90, 2, 1, 64), (1, 3, 0, 2, 2, 8),
                                  (0, 3, 5, 2, 2, 8), (1, 0, 5, 2, 1, 8)):
        q, k, v, do = n(B, Lq, Hq, D), n(B, Lk, Hkv, D), n(B, Lk, Hkv, D), n(B, Lq, Hq, D)
        tab, lens, keep = n(16, Hq), rs.randint(0, Lk + 2, B), rs.rand(B, Lk) < 0.7
        for kw in ({}, dict(scale=0.3, causal=True, q_offset=4), dict(kv_lens=lens, key_mask=keep, bias=tab, q_offset=-2)):
            th = {x: up(y) if isinstance(y, np.ndarray) else y for x, y in kw.items()}
            if "bias" in kw:
                kw, th = dict(kw, bias=A.BucketBias(tab, 30, True)), dict(th, bias=A.BucketBias(up(tab), 30, True))
            r = A.attention(up(q), up(k), up(v), **th)
            h = ops.attention(q, k, v, **kw)
            same(h, r)
            same(ops.attention_backward(do, q, k, v, *h, **kw), A.attention_backward(up(do), up(q), up(k), up(v), *r, **th))
        b, bt = A.BucketBias(tab, 30, False), A.BucketBias(up(tab), 30, False)
        same(ops.relative_bias(b, Lq, Lk, 3), A.relative_bias(bt, Lq, Lk, q_offset=3))
        d = n(B, Hq, Lq, Lk)
        same(ops.relative_bias_backward(b, d, 3), A.relative_bias_backward(bt, up(d), q_offset=3))
    for B, L, Hq, Hk, D, R in ((2, 5, 4, 2, 64, 64), (1, 9, 3, 0, 18, 6), (0, 4, 1, 1, 8, 8), (2, 3, 1, 1, 32, 0)):
        q, k, gq, gk, ang = n(B, L, Hq, D), n(B, L, Hk, D), n(B, L, Hq, D), n(B, L, Hk, D), n(20, R // 2)
        x = (q, k, n(D), n(D), np.cos(ang), np.sin(ang))
        for kw in ({}, dict(positions=rs.randint(0, 20, (B, L)), interleaved=True, eps=1e-3), dict(positions=rs.randint(0, 20, L))):
            th = {a: up(y) if isinstance(y, np.ndarray) else y for a, y in kw.items()}
            same(ops.qk_norm_rope(*x, **kw), A.qk_norm_rope(*map(up, x), **th))
            same(ops.qk_norm_rope_backward(gq, gk, *x, **kw), A.qk_norm_rope_backward(up(gq), up(gk), *map(up, x), **th))
