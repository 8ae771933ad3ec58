"""Attention operators in 64 bits, from their definitions (the oracle of
``rvc_cuda.attention``): plain numpy, one head at a time."""

from __future__ import annotations

import math

import numpy as np


def bucket(rel, num_buckets, max_distance, bidirectional):
    """Bucket of every relative position (key minus query) of the array ``rel``."""
    rel = np.asarray(rel, np.int64)
    n = num_buckets // 2 if bidirectional else num_buckets
    e = n // 2
    a = np.abs(rel) if bidirectional else np.maximum(-rel, 0)
    # a distance on a border (within 1e-9 of a whole number) belongs behind it
    y = np.log(np.maximum(a, 1) / e) / math.log(max_distance / e) * (n - e)
    far = np.minimum(e + np.floor(y + 1e-9).astype(np.int64), n - 1)
    b = np.where(a < e, a, far)
    return np.where(rel > 0, b + n, b) if bidirectional else b


def alive(B, Lq, Lk, kv_lens=None, key_mask=None, causal=False, q_offset=0):
    """[B, Lq, Lk]: the pairs that take part."""
    j = np.arange(Lk)
    a = np.ones((B, Lq, Lk), bool)
    if kv_lens is not None:
        a &= (j < np.asarray(kv_lens)[:, None])[:, None]
    if key_mask is not None:
        a &= np.asarray(key_mask, bool)[:, None]
    if causal:
        a &= j <= np.arange(Lq)[:, None] + q_offset
    return a


def scores(q, k, scale, live, bias=None):
    """Scaled scores [B, Hq, Lq, Lk] with dead pairs at -inf; dead keys are read
    as zeros.  ``bias`` [Hq, Lq, Lk]."""
    q, k = np.asarray(q, np.float64), np.asarray(k, np.float64)
    k = np.where(live.any(1)[:, :, None, None], k, 0.0)
    g = q.shape[2] // k.shape[2]
    s = np.einsum("bihd,bjhd->bhij", q, np.repeat(k, g, 2)) * scale
    if bias is not None:
        s = s + np.asarray(bias, np.float64)
    return np.where(live[:, None], s, -np.inf)


def softmax(s):
    """(p, lse) over the last axis; a row of -inf gives zeros and -inf."""
    if s.shape[-1] == 0:
        return np.zeros_like(s), np.full(s.shape[:-1], -np.inf)
    m = s.max(-1, keepdims=True)
    m0 = np.where(np.isfinite(m), m, 0.0)
    x = np.exp(s - m0)
    t = x.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (m0 + np.log(t))[..., 0]
    return x / np.where(t > 0, t, 1.0), lse


def clean(x, live):
    """Keys or values with what is dead for every query read as zeros."""
    return np.where(live.any(1)[:, :, None, None], np.asarray(x, np.float64), 0.0)


def attention(q, k, v, scale, live, bias=None):
    p, lse = softmax(scores(q, k, scale, live, bias))
    g = q.shape[2] // k.shape[2]
    return np.einsum("bhij,bjhd->bihd", p, np.repeat(clean(v, live), g, 2)), lse, p


def attention_backward(dout, q, k, v, scale, live, bias=None, buckets=None, num_buckets=0):
    """(dq, dk, dv, dtable, p, dp, ds); ``buckets [Lq, Lk]`` of the pairs."""
    q, dout = np.asarray(q, np.float64), np.asarray(dout, np.float64)
    k0, v0 = clean(k, live), clean(v, live)
    B, Lk, Hkv, D = k0.shape
    g = q.shape[2] // Hkv
    p, _ = softmax(scores(q, k, scale, live, bias))
    dp = np.einsum("bihd,bjhd->bhij", dout, np.repeat(v0, g, 2))
    ds = p * (dp - (p * dp).sum(-1, keepdims=True))
    dq = np.einsum("bhij,bjhd->bihd", ds, np.repeat(k0, g, 2)) * scale
    dk = (np.einsum("bhij,bihd->bjhd", ds, q) * scale).reshape(B, Lk, Hkv, g, D).sum(3)
    dv = np.einsum("bhij,bihd->bjhd", p, dout).reshape(B, Lk, Hkv, g, D).sum(3)
    dt = None
    if buckets is not None:
        dt = np.zeros((num_buckets, q.shape[2]))
        for h in range(q.shape[2]):
            np.add.at(dt[:, h], buckets, ds[:, h].sum(0))
    return dq, dk, dv, dt, p, dp, ds


def norm_rope(x, w, cos, sin, positions, eps, interleaved):
    """One of q and k: x [B, L, H, D], positions [B, L]."""
    x = np.asarray(x, np.float64)
    R = 2 * cos.shape[1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    c, s = (np.asarray(t, np.float64)[positions][:, :, None] for t in (cos, sin))
    i = np.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out = y.copy()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., a] * s + y[..., b] * c
    return out


def norm_rope_backward(dy, x, w, cos, sin, positions, eps, interleaved):
    x, dy, w = (np.asarray(t, np.float64) for t in (x, dy, w))
    D, R = x.shape[-1], 2 * cos.shape[1]
    c, s = (np.asarray(t, np.float64)[positions][:, :, None] for t in (cos, sin))
    i = np.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    g = dy.copy()
    g[..., a] = dy[..., a] * c + dy[..., b] * s
    g[..., b] = dy[..., b] * c - dy[..., a] * s
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dw = (g * x * r).sum((0, 1, 2))
    gw = g * w
    return r * gw - x * r ** 3 * (gw * x).sum(-1, keepdims=True) / D, dw
