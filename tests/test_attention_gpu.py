"""Attention operators on the GPU against the 64-bit oracle, element by element.

Tolerances follow from the roundings of the kernels, none is fitted.  With
u = half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24):

* a score carries the error ds = 2^-20 sum_d |q_d k_d| |scale| + 2^-21 |s| (fp32
  operands split in two TF32 parts: 2^-22 for each of the dropped and rounded
  parts, fp32 sums) - for 16-bit inputs the products are exact and the same
  bound covers the fp32 sums;
* a weight p then has the relative error 2 ds + 2^-20 (its own score and the
  row's log sum; ex2 and the sum), and w = u (16 bits) or 2^-20 (fp32) when it
  is rounded for its second product;
* out: u |out| + sum_j p |v| (2 ds + 2^-20 + w);
* dS = p (dP - delta): p ((|dP| + |delta|) (2 ds + 2^-20) + 2^-20 sum |do v| +
  sum |do| u |out|) (delta is formed with the rounded output), plus w |dS| when
  it is rounded; the gradients' own rounding is u of their value.  A type's
  smallest step is added once per rounding: 2^-25 for fp16's subnormals, and
  2^-120 for the others (a weight below 2^-126 is flushed to zero, and it
  multiplies values and gradients below 2^6).
"""

import numpy as np
import pytest
import torch

from oracle import attention as OA

pytestmark = pytest.mark.gpu

from rvc_cuda import _lib, attention as A, ops  # noqa: E402

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -120


def f8(x):
    return x.double().cpu().numpy()


def rnd(rs, t, *shape, scale=1.0):
    return torch.from_numpy(rs.standard_normal(shape) * scale).to("cuda", t)


def close(got, want, tol, what):
    got = f8(got)
    assert got.shape == want.shape, what
    same = np.isneginf(want)
    np.testing.assert_array_equal(np.isneginf(got), same, err_msg=what)
    d = np.abs(np.where(same, 0.0, got) - np.where(same, 0.0, want))
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(d / np.maximum(tol, 1e-300)):.3g} x the bound"


class Case:
    """Inputs of one attention call and what the oracle says of it."""

    def __init__(self, dtype, B, Hq, Hkv, D, Lq, Lk, seed=0, lens=None, keep=None, causal=False, q_offset=0, bias=None,
                 junk=None, scale=None, packed=False, lens_type=torch.int32):
        rs = np.random.RandomState(seed)
        t = self.t = DT[dtype]
        self.scale = scale if scale is not None else 1.0 / np.sqrt(D)
        if packed:  # parts of one projection, and a broadcast batch of queries
            kv = rnd(rs, t, B, Lk, 2, Hkv, D)
            k, v = kv[:, :, 0], kv[:, :, 1]
            q = rnd(rs, t, 1, Hq, Lq, D).transpose(1, 2).expand(B, Lq, Hq, D)
        else:
            q, k, v = rnd(rs, t, B, Lq, Hq, D), rnd(rs, t, B, Lk, Hkv, D), rnd(rs, t, B, Lk, Hkv, D)
        self.kw = {"causal": causal, "q_offset": q_offset, "scale": scale}
        cut = None
        if lens is not None:
            self.kw["kv_lens"] = torch.tensor(lens, device="cuda", dtype=lens_type)
            cut = np.clip(lens, 0, Lk)
        if keep == "random":
            keep = rs.rand(B, Lk) < 0.6
            keep[0] = False  # a batch entry with nothing to see
        if keep is not None:
            self.kw["key_mask"] = torch.from_numpy(np.asarray(keep)).cuda()
        self.live = OA.alive(B, Lq, Lk, cut, keep, causal, q_offset)
        if junk is not None:  # what padding may hold
            dead = torch.from_numpy(~OA.alive(B, 1, Lk, cut, keep)[:, 0]).cuda()
            k, v = k.masked_fill(dead[:, :, None, None], junk), v.masked_fill(dead[:, :, None, None], junk)
        self.q, self.k, self.v = q, k, v
        self.where = self.tab = None
        self.n = 0
        if bias is not None:
            self.n, far, both = bias
            tab = rnd(rs, t, self.n, Hq)
            self.kw["bias"] = A.BucketBias(tab, far, both)
            self.where = OA.bucket(np.arange(Lk)[None] - np.arange(Lq)[:, None] - q_offset, self.n, far, both)
            self.tab = f8(tab).T[:, self.where]
        self.do = rnd(rs, t, B, Lq, Hq, D)
        q, k, v = f8(q), OA.clean(f8(k), self.live), OA.clean(f8(v), self.live)
        self.q8, self.k8, self.v8 = q, k, v
        self.g = Hq // Hkv
        self.out, self.lse, self.p = OA.attention(q, k, v, self.scale, self.live, self.tab)
        u = half_step(t)
        self.w = u if t != torch.float32 else 2.0 ** -20
        rep = lambda x: np.repeat(x, self.g, 2)  # noqa: E731
        mag = np.einsum("bihd,bjhd->bhij", np.abs(q), rep(np.abs(k))) * abs(self.scale)
        s = OA.scores(q, k, self.scale, self.live, self.tab)
        self.es = np.where(np.isfinite(s), 2.0 ** -20 * mag + 2.0 ** -21 * np.abs(np.where(np.isfinite(s), s, 0)), 0.0)
        self.ep = 2 * self.es.max(-1, keepdims=True, initial=0.0) + 2.0 ** -20  # relative error of a weight
        self.pv = np.einsum("bhij,bjhd->bihd", self.p * (self.ep + self.w), rep(np.abs(v)))

    def forward(self):
        out, lse = A.attention(self.q, self.k, self.v, **self.kw)
        u = half_step(self.t)
        close(out, self.out, u * np.abs(self.out) + self.pv + tiny(self.t) * (2 + self.live.shape[2]), "out")
        lim = self.es.max(-1, initial=0.0) + 2.0 ** -20 + 2.0 ** -22 * np.abs(np.where(np.isfinite(self.lse), self.lse, 0))
        close(lse, self.lse, lim, "lse")
        return out, lse

    def backward(self):
        t, u, w = self.t, half_step(self.t), self.w
        out = torch.from_numpy(self.out).to("cuda", t)
        lse = torch.from_numpy(self.lse).to("cuda", torch.float32)
        got = A.attention_backward(self.do, self.q, self.k, self.v, out, lse, **self.kw)
        do = f8(self.do)
        dq, dk, dv, dt, p, dp, ds = OA.attention_backward(do, self.q8, self.k8, self.v8, self.scale, self.live,
                                                          self.tab, self.where, self.n)
        rep = lambda x: np.repeat(x, self.g, 2)  # noqa: E731
        fold = lambda x: x.reshape(x.shape[0], x.shape[1], -1, self.g, x.shape[3]).sum(3)  # noqa: E731
        delta = (p * dp).sum(-1, keepdims=True)
        edelta = np.einsum("bihd,bihd->bhi", np.abs(do), np.abs(self.out))[..., None] * (u + 2.0 ** -22)
        ep = self.ep + 2.0 ** -24 * np.abs(np.where(np.isfinite(self.lse), self.lse, 0))[..., None]  # lse came rounded
        mag = np.einsum("bihd,bjhd->bhij", np.abs(do), rep(np.abs(self.v8)))
        eds = p * ((np.abs(dp) + np.abs(delta)) * ep + 2.0 ** -20 * mag + edelta)
        rds = eds + w * np.abs(ds) + tiny(t)  # as it enters dq and dk
        small = tiny(t)
        close(got[2], dv, u * np.abs(dv) + fold(np.einsum("bhij,bihd->bjhd", p * (ep + w) + small, np.abs(do))) + small, "dv")
        close(got[0], dq, u * np.abs(dq) + np.einsum("bhij,bjhd->bihd", rds + 2.0 ** -20 * np.abs(ds), rep(np.abs(self.k8)))
              * abs(self.scale) + small, "dq")
        close(got[1], dk, u * np.abs(dk) + fold(np.einsum("bhij,bihd->bjhd", rds + 2.0 ** -20 * np.abs(ds), np.abs(self.q8)))
              * abs(self.scale) + small, "dk")
        if self.where is not None:
            tol = np.zeros_like(dt)
            for h in range(dt.shape[1]):
                np.add.at(tol[:, h], self.where, (eds + 2.0 ** -20 * np.abs(ds))[:, h].sum(0))
            close(got[3], dt, u * np.abs(dt) + tol + small, "dtable")
        return got


SIZES = [  # B, Hq, Hkv, D, Lq, Lk
    (1, 1, 1, 1, 1, 1), (2, 4, 2, 33, 1, 70), (1, 12, 12, 64, 1, 499), (2, 8, 1, 128, 2, 1000), (3, 4, 4, 40, 17, 5),
    (1, 2, 2, 96, 130, 129), (2, 6, 3, 64, 64, 64), (1, 4, 2, 128, 200, 333), (1, 3, 3, 80, 257, 63),
    (2, 2, 1, 24, 65, 257), (1, 2, 2, 64, 384, 640), (1, 1, 1, 128, 300, 300), (33, 2, 2, 32, 3, 9),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(dtype, size):
    Case(dtype, *size).forward()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward(dtype, size):
    Case(dtype, *size).backward()


MASKS = {
    "lens": dict(lens=[0, 70, 129], junk=float("nan")),
    "lens_past_the_end": dict(lens=[1, 10**6, -5], junk=float("inf"), lens_type=torch.int64),
    "keys": dict(keep="random", junk=float("nan")),
    "keys_and_lens": dict(keep="random", lens=[129, 65, 128], junk=float("-inf")),
    "causal": dict(causal=True, q_offset=0),
    "causal_rows_before_the_first_key": dict(causal=True, q_offset=-40),
    "causal_past_all": dict(causal=True, q_offset=500, lens=[129, 3, 64]),
    "causal_lens": dict(causal=True, q_offset=50, lens=[129, 64, 1], junk=float("nan")),
    "bias": dict(bias=(32, 20, True)),
    "bias_one_way_causal": dict(bias=(16, 40, False), causal=True, q_offset=3),
    "bias_offset_lens": dict(bias=(320, 800, True), q_offset=77, lens=[129, 100, 0]),
    "bias_far_offset": dict(bias=(8, 6, True), q_offset=-(1 << 31) + 5),
    "scale_packed": dict(scale=0.02, packed=True),
    "negative_scale": dict(scale=-0.3, keep="random"),
    "large_scores": dict(scale=40.0),
}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("Lq", [1, 150])
def test_masks_and_bias(dtype, mask, Lq):
    c = Case(dtype, 3, 4, 2, 64, Lq, 129, **MASKS[mask])
    c.forward()
    c.backward()


SPLIT = {
    "plain": {},
    "lens": dict(lens=[4100, 0], junk=float("nan")),
    "keys_bias": dict(keep="random", bias=(32, 400, True), junk=float("inf")),
    "causal": dict(causal=True, q_offset=700),
    "causal_nothing": dict(causal=True, q_offset=-100000),
}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("mask", SPLIT, ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_keys_split_over_blocks(dtype, mask, D):
    """Few queries on long states: the keys are shared out to blocks and joined,
    on every path (few rows, many rows, tensor-core tiles), some shares empty."""
    for Lq in (2, 40, 130):
        Case(dtype, 2, 2, 1, D, Lq, 4100, **SPLIT[mask]).forward()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [40, 128])
def test_shares_of_a_group(dtype, D):
    """Few key tiles and a large group: its query heads are shared out to blocks."""
    Case(dtype, 1, 7, 1, D, 150, 200, bias=(32, 60, True), causal=True, q_offset=50).backward()
    Case(dtype, 3, 24, 2, D, 70, 300, lens=[300, 0, 129], junk=float("nan"), bias=(16, 30, False)).backward()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_causal_with_nothing_alive_and_scale_zero(dtype):
    for kw in (dict(causal=True, q_offset=-100000), dict(scale=0.0), dict(scale=0.0, keep="random", junk=float("nan"))):
        c = Case(dtype, 2, 4, 2, 64, 270, 200, **kw)
        c.forward()
        c.backward()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_bias_gradient_over_many_tiles(dtype, D):
    """Near and far diagonals, lengths that are no multiple of a tile, two batch entries."""
    for bias, kw in (((32, 128, True), {}), ((64, 300, False), dict(causal=True, q_offset=130))):
        Case(dtype, 2, 2, 1, D, 515, 645, bias=bias, **kw).backward()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_queries_with_one_key(dtype):
    """A softmax over one key is 1: no gradient reaches q, k or the table, exactly."""
    for Lq, Lk, kw in ((1, 1, {}), (70, 1, {}), (5, 40, dict(lens=[1, 1])), (1, 9, dict(causal=True))):
        c = Case(dtype, 2, 4, 2, 64, Lq, Lk, bias=(8, 6, True), **kw)
        dq, dk, _, dt = c.backward()
        assert (dq == 0).all() and (dk == 0).all() and (dt == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_no_keys_and_no_rows(dtype):
    c = Case(dtype, 2, 4, 2, 64, 7, 0, bias=(8, 6, True))
    out, lse = c.forward()
    assert (out == 0).all() and torch.isneginf(lse).all()
    dq, dk, dv, dt = A.attention_backward(c.do, c.q, c.k, c.v, out, lse, **c.kw)
    assert (dq == 0).all() and dk.shape == (2, 0, 2, 64) and (dt == 0).all()
    for B, Lq in ((2, 0), (0, 3)):
        c = Case(dtype, B, 4, 2, 64, Lq, 5)
        out, lse = A.attention(c.q, c.k, c.v)
        assert out.shape == (B, Lq, 4, 64) and lse.shape == (B, 4, Lq)
        dq, dk, dv = A.attention_backward(c.do, c.q, c.k, c.v, out, lse)
        assert (dk == 0).all() and (dv == 0).all() and dq.shape == (B, Lq, 4, 64)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_unaligned_and_transposed_inputs(dtype):
    """Starts and strides that no wide load may touch, and a head's values apart."""
    for D, pad in ((64, 1), (64, 3), (72, 4), (128, 2)):
        c = Case(dtype, 2, 2, 2, D, 70, 90)

        def off(x):
            y = torch.empty((*x.shape[:3], D + pad), device="cuda", dtype=x.dtype).fill_(float("nan"))
            y[..., pad:] = x
            return y[..., pad:]

        c.q, c.k, c.v, c.do = off(c.q), off(c.k), off(c.v), off(c.do)
        c.forward()
        c.backward()
        c.k = c.k.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
        c.forward()
        c.backward()


def test_offsets_past_32_bits():
    """Two batch entries of a cache whose second lies more than 2^31 elements on."""
    far = (1 << 31) + 4096
    store = torch.zeros(far + 300 * 64 * 2, device="cuda", dtype=torch.bfloat16)
    c = Case("bf16", 2, 2, 2, 64, 150, 300, lens=[300, 170])
    k = store.as_strided((2, 300, 2, 64), (far, 128, 64, 1))
    k.copy_(c.k)
    c.k = k
    c.forward()
    c.backward()
    c.q = c.q[:, :1]
    out, _ = A.attention(c.q, c.k, c.v, kv_lens=c.kw["kv_lens"])
    close(out, c.out[:, :1], half_step(torch.bfloat16) * np.abs(c.out[:, :1]) + c.pv[:, :1], "one row")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_same_call_same_bits(dtype):
    for size in ((2, 4, 2, 64, 1, 3000), (2, 4, 2, 128, 300, 500)):
        c = Case(dtype, *size, bias=(32, 100, True), lens=[size[5], 200])
        a = [*A.attention(c.q, c.k, c.v, **c.kw), *c.backward()]
        for _ in range(3):
            b = [*A.attention(c.q, c.k, c.v, **c.kw), *c.backward()]
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_streams_and_graphs(dtype):
    """Two calls in flight on two streams, and two captured graphs replayed on
    new inputs, give what single calls give."""
    cs = [Case(dtype, 2, 4, 2, 64, L, 700, seed=s, bias=(32, 100, True), lens=[700, 300])
          for s, L in ((1, 1), (2, 260))]
    want = [[x.clone() for x in (*A.attention(c.q, c.k, c.v, **c.kw), *c.backward())] for c in cs]
    o = [torch.from_numpy(c.out).to("cuda", c.t) for c in cs]
    z = [torch.from_numpy(c.lse).to("cuda", torch.float32) for c in cs]
    torch.cuda.synchronize()

    def both(n, q=None):
        c = cs[n]
        q = c.q if q is None else q
        return [*A.attention(q, c.k, c.v, **c.kw), *A.attention_backward(c.do, q, c.k, c.v, o[n], z[n], **c.kw)]

    ss = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        got = []
        for n, s in enumerate(ss):
            with torch.cuda.stream(s):
                got.append(both(n))
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(x, y))
    graphs, outs, qs = [], [], [torch.zeros_like(c.q) for c in cs]
    for n, s in enumerate(ss):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(both(n, qs[n]))
        graphs.append(g)
    for n, c in enumerate(cs):
        qs[n].copy_(c.q)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, ss):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, outs):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


# ------------------------------------------------------------ bias as a tensor


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", [(1, 1, 1), (3, 7, 300), (2, 499, 257), (12, 33, 1024), (2, 1025, 31)], ids=str)
@pytest.mark.parametrize("bias,off", [((32, 128, True), 0), ((6, 50, False), -3), ((320, 800, True), 400)])
def test_relative_bias(dtype, size, bias, off):
    H, Lq, Lk = size
    rs, t = np.random.RandomState(3), DT[dtype]
    n, far, both = bias
    b = A.BucketBias(rnd(rs, t, n, H), far, both)
    where = OA.bucket(np.arange(Lk)[None] - np.arange(Lq)[:, None] - off, n, far, both)
    got = A.relative_bias(b, Lq, Lk, q_offset=off)
    assert got.dtype == t
    np.testing.assert_array_equal(f8(got), f8(b.table).T[:, where])  # values are copied
    d = rnd(rs, t, 2, H, Lq, Lk + 3)[..., 1:Lk + 1]  # rows that are not aligned
    want, mag = np.zeros((n, H)), np.zeros((n, H))
    for h in range(H):
        np.add.at(want[:, h], where, f8(d)[:, h].sum(0))
        np.add.at(mag[:, h], where, np.abs(f8(d))[:, h].sum(0))
    # fp32 sums of at most 300 addends along a diagonal's part, 2^-24 each, then 64 bits and one rounding
    tol = half_step(t) * np.abs(want) + 300 * 2.0 ** -24 * mag + tiny(t)
    close(A.relative_bias_backward(b, d, q_offset=off), want, tol, "dtable")
    close(A.relative_bias_backward(b, d[0], q_offset=off).float() + A.relative_bias_backward(b, d[1], q_offset=off).float(),
          want, 2 * half_step(t) * (mag + np.abs(want)) + 300 * 2.0 ** -24 * mag + 2 * tiny(t), "dtable in two calls")


def test_relative_bias_without_pairs():
    b = A.BucketBias(torch.ones(8, 3, device="cuda"), 6, True)
    assert A.relative_bias(b, 0, 5).shape == (3, 0, 5) and A.relative_bias(b, 4, 0).shape == (3, 4, 0)
    assert (A.relative_bias_backward(b, torch.ones(2, 3, 0, 5, device="cuda")) == 0).all()


def test_relative_bias_broadcast_gradient():
    """A gradient with stride 0 over the batch and the rows."""
    b = A.BucketBias(torch.zeros(8, 2, device="cuda"), 6, True)
    d = torch.arange(2 * 9, device="cuda", dtype=torch.float32).reshape(1, 2, 1, 9).expand(5, 2, 11, 9)
    np.testing.assert_allclose(f8(A.relative_bias_backward(b, d)), f8(A.relative_bias_backward(b, d.contiguous())),
                               rtol=0, atol=0)


def test_attention_with_the_bias_is_attention_with_its_tensor():
    """The bias inside the softmax equals scores with ``relative_bias`` added, and
    their table gradients agree: both sides are exact up to fp32 sums."""
    c = Case("fp32", 2, 4, 4, 64, 200, 230, bias=(32, 100, True), q_offset=9)
    t = f8(A.relative_bias(c.kw["bias"], 200, 230, q_offset=9))
    np.testing.assert_array_equal(t, c.tab)
    dq, dk, dv, dt = c.backward()
    _, _, _, _, _, _, ds = OA.attention_backward(f8(c.do), c.q8, c.k8, c.v8, c.scale, c.live, c.tab)
    via = A.relative_bias_backward(c.kw["bias"], torch.from_numpy(ds).to("cuda", torch.float32), q_offset=9)
    scale = np.abs(ds).sum((0, 2, 3)).max()
    close(dt, f8(via), np.full(dt.shape, 2.0 ** -17 * scale), "dtable both ways")


# ---------------------------------------------------------- norm and rotation

ROPE = [  # B, L, Hq, Hk, D, R
    (1, 1, 1, 1, 2, 2), (2, 5, 4, 2, 64, 64), (3, 1, 16, 4, 128, 128), (1, 130, 3, 3, 96, 96), (2, 33, 2, 1, 128, 64),
    (2, 9, 5, 1, 40, 24), (1, 17, 2, 2, 18, 6), (2, 70, 1, 1, 256, 128), (1, 7, 4, 0, 64, 64), (1, 50, 2, 2, 32, 0),
    (4, 700, 8, 2, 64, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", ROPE, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_norm_rope(dtype, size, interleaved):
    B, L, Hq, Hk, D, R = size
    rs, t = np.random.RandomState(5), DT[dtype]
    qkv = rnd(rs, t, B, L, Hq + 2 * Hk, D, scale=1.5)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    wt = t if D == 64 else torch.float32
    wq, wk = 1 + rnd(rs, wt, D, scale=0.2), 1 + rnd(rs, wt, D, scale=0.2)
    cos, sin = A.rope_table(1000, R, device="cuda") if R else (torch.zeros(1000, 0, device="cuda"),) * 2
    pos = rs.randint(0, 1000, (B, L))
    p = torch.from_numpy(pos).cuda()
    how = dict(positions=p if L % 2 else p.int(), eps=1e-5, interleaved=interleaved)
    u, small = half_step(t), tiny(t)
    got = A.qk_norm_rope(q, k, wq, wk, cos, sin, **how)
    dqo, dko = rnd(rs, t, B, L, Hq, D), rnd(rs, t, B, L, Hk, D)
    grads = A.qk_norm_rope_backward(dqo, dko, q, k, wq, wk, cos, sin, **how)
    for n, (x, w, dy) in enumerate(((q, wq, dqo), (k, wk, dko))):
        if x.shape[2] == 0:
            assert got[n].shape == x.shape and (grads[2 + n] == 0).all()
            continue
        y = OA.norm_rope(f8(x), f8(w), f8(cos), f8(sin), pos, 1e-5, interleaved)
        # fp32 on the way: a pair's two products, each to 2^-20 (norm, weight, turn)
        m = np.abs(f8(x)) / np.sqrt((f8(x) ** 2).mean(-1, keepdims=True)) * np.abs(f8(w))
        pair = m.max(-1, keepdims=True)
        close(got[n], y, u * np.abs(y) + 2.0 ** -20 * pair + small, f"output {n}")
        dx, dw = OA.norm_rope_backward(f8(dy), f8(x), f8(w), f8(cos), f8(sin), pos, 1e-5, interleaved)
        r = 1 / np.sqrt((f8(x) ** 2).mean(-1, keepdims=True) + 1e-5)
        g = np.abs(f8(dy)).max(-1, keepdims=True) * np.abs(f8(w)).max() * 2
        lim = r * g * (1 + (np.abs(f8(x)) * r).max(-1, keepdims=True) ** 2)
        close(grads[n], dx, u * np.abs(dx) + 2.0 ** -20 * lim + small, f"input gradient {n}")
        gw = (np.abs(f8(dy)).max(-1, keepdims=True) * 2 * np.abs(f8(x)) * r).sum((0, 1, 2))
        uw = half_step(wt)
        # at most 2^12 addends of a lane in 32 bits, 2^-24 each in the worst order, 64 bits beyond
        rows = min(4096, B * L * x.shape[2])
        close(grads[2 + n], dw, uw * np.abs(dw) + (2.0 ** -20 + rows * 2.0 ** -24) * gw + tiny(wt), f"weight gradient {n}")


def test_norm_rope_positions():
    """Default and broadcast positions; a position outside the tables gives NaN there and nowhere else."""
    rs = np.random.RandomState(6)
    q, k, w = rnd(rs, torch.float32, 2, 6, 2, 32), rnd(rs, torch.float32, 2, 6, 1, 32), torch.ones(32, device="cuda")
    cos, sin = A.rope_table(40, 32, device="cuda")
    a = A.qk_norm_rope(q, k, w, w, cos, sin)
    b = A.qk_norm_rope(q, k, w, w, cos, sin, positions=torch.arange(6, device="cuda"))
    c = A.qk_norm_rope(q, k, w, w, cos, sin, positions=torch.arange(6, device="cuda").expand(2, 6))
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    pos = torch.arange(6, device="cuda").repeat(2, 1)
    pos[0, 2], pos[1, 5] = 40, -1
    d = A.qk_norm_rope(q, k, w, w, cos, sin, positions=pos)
    for x, y in zip(a, d):
        bad = torch.isnan(y).all(-1).all(-1)
        assert bad.nonzero().tolist() == [[0, 2], [1, 5]]
        assert torch.equal(x[~bad], y[~bad])


def test_zero_rows_of_norm_rope():
    """A head of zeros stays zero; its gradient is finite."""
    q, w = torch.zeros(1, 2, 1, 64, device="cuda"), torch.ones(64, device="cuda")
    cos, sin = A.rope_table(2, 64, device="cuda")
    y, _ = A.qk_norm_rope(q, q, w, w, cos, sin)
    assert (y == 0).all()
    g = A.qk_norm_rope_backward(torch.ones_like(q), torch.ones_like(q), q, q, w, w, cos, sin)
    assert all(torch.isfinite(x).all() for x in g)
    e = torch.empty(0, 2, 1, 64, device="cuda")
    g = A.qk_norm_rope_backward(e, e, e, e, w, w, cos, sin)
    assert (g[2] == 0).all() and (g[3] == 0).all()


# -------------------------------------------------------------- used together


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_block_of_both_attentions(dtype):
    """A decoder block's use: norm and rotation, causal self attention with the
    bias, then attention to encoder states of another length - forward, and the
    chain of the three backward passes, against the oracle's chain in 64 bits."""
    rs, t = np.random.RandomState(7), DT[dtype]
    B, L, Le, H, Hk, D = 2, 140, 210, 4, 2, 64
    qkv = rnd(rs, t, B, L, H + 2 * Hk, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    enc = rnd(rs, t, B, Le, 2, Hk, D)
    w = 1 + rnd(rs, torch.float32, D, scale=0.1)
    cos, sin = A.rope_table(L, D, device="cuda")
    bias = A.BucketBias(rnd(rs, t, 32, H), 64, False)
    lens = torch.tensor([Le, 77], device="cuda")
    do = rnd(rs, t, B, L, H, D)
    qn, kn = A.qk_norm_rope(q, k, w, w, cos, sin)
    x, z1 = A.attention(qn, kn, v, causal=True, bias=bias)
    y, z2 = A.attention(x, enc[:, :, 0], enc[:, :, 1], kv_lens=lens)
    dx, dek, dev = A.attention_backward(do, x, enc[:, :, 0], enc[:, :, 1], y, z2, kv_lens=lens)
    dqn, dkn, dv, dt = A.attention_backward(dx, qn, kn, v, x, z1, causal=True, bias=bias)
    dq, dk, dwq, dwk = A.qk_norm_rope_backward(dqn, dkn, q, k, w, w, cos, sin)

    pos = np.broadcast_to(np.arange(L), (B, L))
    args = (f8(w), f8(cos), f8(sin), pos, 1e-6, False)
    oq, ok = OA.norm_rope(f8(q), *args), OA.norm_rope(f8(k), *args)
    live1, live2 = OA.alive(B, L, L, causal=True), OA.alive(B, L, Le, kv_lens=[Le, 77])
    where = OA.bucket(np.arange(L)[None] - np.arange(L)[:, None], 32, 64, False)
    tab = f8(bias.table).T[:, where]
    ox = OA.attention(oq, ok, f8(v), 0.125, live1, tab)[0]
    e = f8(enc)
    oy = OA.attention(ox, e[:, :, 0], e[:, :, 1], 0.125, live2)[0]
    odx, odek, odev = OA.attention_backward(f8(do), ox, e[:, :, 0], e[:, :, 1], 0.125, live2)[:3]
    odq, odk, odv, odt = OA.attention_backward(odx, oq, ok, f8(v), 0.125, live1, tab, where, 32)[:4]
    fq, fwq = OA.norm_rope_backward(odq, f8(q), *args)
    fk, fwk = OA.norm_rope_backward(odk, f8(k), *args)
    # 2-norms over whole tensors: a chain of at most eight tensors and sixteen
    # weights rounded to the type, each adding at most u of the norm where scores
    # stay of order one (no error grows: |d score| <= |q| |k| / 8 u ~ 8 u)
    lim = 32 * half_step(t) if t != torch.float32 else 2.0 ** -16
    for n, (a, b) in {"y": (y, oy), "dq": (dq, fq), "dk": (dk, fk), "dv": (dv, odv), "dtable": (dt, odt),
                      "dek": (dek, odek), "dev": (dev, odev), "dwq": (dwq, fwq), "dwk": (dwk, fwk)}.items():
        assert np.linalg.norm(f8(a) - b) <= lim * np.linalg.norm(b), n


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradients_against_differences(dtype):
    """Central differences of the kernel's own forward pass along a random
    direction of each input (fp32; the 16-bit case checks the fp32 call on the
    same values)."""
    c = Case("fp32", 2, 4, 2, 32, 70, 90, bias=(16, 40, True), lens=[90, 33])
    if dtype == "bf16":
        c.q, c.k, c.v = (x.bfloat16().float() for x in (c.q, c.k, c.v))
    out, lse = A.attention(c.q, c.k, c.v, **c.kw)
    got = A.attention_backward(c.do, c.q, c.k, c.v, out, lse, **c.kw)
    rs = np.random.RandomState(8)
    tab = c.kw["bias"].table

    def loss(q, k, v, t):
        kw = dict(c.kw, bias=A.BucketBias(t, 40, True))
        return float((A.attention(q, k, v, **kw)[0].double() * c.do.double()).sum())

    args = [c.q, c.k, c.v, tab]
    for n in range(4):
        d = rnd(rs, torch.float32, *args[n].shape)
        d /= d.norm()
        h = 2.0 ** -5
        hi, lo = list(args), list(args)
        hi[n], lo[n] = args[n] + h * d, args[n] - h * d
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        want = float((got[n].double() * d.double()).sum())
        # third derivatives along a unit direction are below 2 |do| |v| ~ 500: h^2 / 6 of that; the
        # differences' own rounding is 2^-20 |do| |out| / h ~ 0.01
        assert abs(diff - want) <= 500 * h * h / 6 + 0.02, (n, diff, want)


# ------------------------------------------------------------------ host forms


def test_numpy_forms():
    rs = np.random.RandomState(9)
    q, k, v = (rs.standard_normal(s).astype(np.float32) for s in ((2, 30, 4, 32), (2, 41, 2, 32), (2, 41, 2, 32)))
    tab = rs.standard_normal((16, 4)).astype(np.float32)
    bias = A.BucketBias(tab, 30, True)
    lens, keep = np.array([41, 20]), rs.rand(2, 41) < 0.8
    out, lse = ops.attention(q, k, v, kv_lens=lens, key_mask=keep, bias=bias)
    live = OA.alive(2, 30, 41, lens, keep)
    where = OA.bucket(np.arange(41)[None] - np.arange(30)[:, None], 16, 30, True)
    o, z, _ = OA.attention(q, k, v, 32 ** -0.5, live, tab.T[:, where])
    # unit-scale scores and values: the element bounds of the module's head, about 2^-17
    np.testing.assert_allclose(out, o, rtol=0, atol=2.0 ** -15)
    np.testing.assert_allclose(lse, z, rtol=0, atol=2.0 ** -15)
    do = rs.standard_normal(q.shape).astype(np.float32)
    got = ops.attention_backward(do, q, k, v, out, lse, kv_lens=lens, key_mask=keep, bias=bias)
    want = OA.attention_backward(do, q, k, v, 32 ** -0.5, live, tab.T[:, where], where, 16)
    for a, b in zip(got, want):
        np.testing.assert_allclose(a, b, rtol=0, atol=2.0 ** -13 * max(1.0, np.abs(b).max()))
    np.testing.assert_array_equal(ops.relative_bias(bias, 30, 41), tab.T[:, where])
    d = rs.standard_normal((4, 30, 41)).astype(np.float32)
    w = np.zeros((16, 4))
    for h in range(4):
        np.add.at(w[:, h], where, d[h])
    np.testing.assert_allclose(ops.relative_bias_backward(bias, d), w, rtol=0, atol=2.0 ** -24 * 300 * 100)
    g = np.ones(32, np.float32)
    cos, sin = (x.numpy() for x in A.rope_table(41, 32, device="cpu"))
    a, b = ops.qk_norm_rope(k, v, g, g, cos, sin)
    pos = np.broadcast_to(np.arange(41), (2, 41))
    np.testing.assert_allclose(a, OA.norm_rope(k, g, cos, sin, pos, 1e-6, False), rtol=0, atol=2.0 ** -17)
    r = ops.qk_norm_rope_backward(a, b, k, v, g, g, cos, sin, positions=pos)
    dx, dw = OA.norm_rope_backward(a, k, g, cos, sin, pos, 1e-6, False)
    np.testing.assert_allclose(r[0], dx, rtol=0, atol=2.0 ** -15)
    np.testing.assert_allclose(r[2], dw, rtol=0, atol=2.0 ** -13 * np.abs(dw).max())
    with pytest.raises(ValueError):
        ops.attention(q, k, v, kv_lens=np.array([1.5, 2.0]))
    with pytest.raises(ValueError):
        ops.attention(q, k[:, :, :, :16], v)


def test_workspace_is_checked():
    """The C entry point refuses a workspace that is too small before any launch."""
    c = Case("bf16", 1, 1, 1, 64, 1, 32768)  # one row on long states: split through the workspace
    desc = (A.C.c_int64 * 29)(1, 1, 1, 1, 1, 32768, 64, *c.q.stride()[:3], *c.k.stride()[:3], *c.v.stride()[:3])
    ctx = _lib.get_context().handle
    need = A.C.c_int64(0)
    _lib.check(_lib.lib.rvc_cuda_attention_workspace(ctx, desc, 29, 0, need))
    assert need.value > 0
    out, lse, ws = torch.empty_like(c.q), torch.empty(1, device="cuda"), torch.empty(need.value, dtype=torch.uint8, device="cuda")
    n0 = _lib.launch_count()

    def call(ws_ptr, nbytes, n=29, lse_ptr=lse.data_ptr()):
        return _lib.lib.rvc_cuda_attention_device(ctx, None, desc, n, 0.125, c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(),
                                                  None, None, None, None, 0, out.data_ptr(), lse_ptr, ws_ptr, nbytes)

    for bad in ((ws.data_ptr(), need.value - 1), (None, need.value), (ws.data_ptr() + 4, need.value)):
        assert call(*bad) == _lib.RVC_E_ARG and "workspace" in _lib.last_error()
    assert call(ws.data_ptr(), need.value, 28) == _lib.RVC_E_ARG
    assert call(ws.data_ptr(), need.value, 29, None) == _lib.RVC_E_ARG
    assert _lib.launch_count() == n0
    assert call(ws.data_ptr(), need.value) == 0
    torch.cuda.synchronize()
