"""Operator module for ``RVC_BACKEND=cuda``.

``runtime.backend`` (``runtime/backend.py:57-70``, ``:189-197``) looks ops up
by name in the registered module and calls them with numpy arrays; each
function here keeps the signature and numpy semantics of the corresponding
``runtime.backend`` wrapper (``runtime/backend.py:205-319``) and returns a new
float32 array.  The math runs in librvc_cuda on the GPU; shapes the library
does not take raise ``ValueError``, which the reference's ``nn`` callers catch
to pick their own path (``runtime/nn.py:286-289``, ``:382-387``, ``:590-593``).

``buf_*`` arguments (the Vulkan engine's resident-buffer handles) are accepted
and ignored.  Nothing here needs torch.
"""

from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._attn_args import MAX_HEAD_DIM, BucketBias, _length, _offset, _pack11, _pack25, _pack29, _scale
from ._lib import check, fptr, iptr, lib

__all__ = [
    "matmul", "add", "mul", "relu", "conv1d", "conv_transpose1d", "embedding",
    "add_inplace", "mul_inplace", "layer_norm", "softmax", "leaky_relu", "gelu",
    "gating", "rel_attention", "im2col_1d", "attention", "attention_backward", "relative_bias",
    "relative_bias_backward", "qk_norm_rope", "qk_norm_rope_backward",
]


def _ctx():
    return _lib.get_context().handle


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a, dtype=np.float32))


def _mm2(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError(f"matmul: shapes {a.shape} and {b.shape} not aligned")
    out = np.empty((M, N), np.float32)
    if M == 0 or N == 0:
        return out
    if K == 0:
        out[:] = 0
        return out
    check(lib.rvc_cuda_matmul(_ctx(), fptr(_f32(a)), fptr(_f32(b)), M, K, N, fptr(out)))
    return out


def matmul(a, b, buf_a=None, buf_b=None):
    """``np.asarray(a) @ np.asarray(b)`` (``runtime/backend.py:205-209``)."""
    a = np.asarray(a)
    b = np.asarray(b)
    if a.ndim == 1 or b.ndim == 1:
        a2 = a[None, :] if a.ndim == 1 else a
        b2 = b[:, None] if b.ndim == 1 else b
        r = matmul(a2, b2)
        if a.ndim == 1:
            r = r[..., 0, :]
        if b.ndim == 1:
            r = r[..., 0]
        return r
    if b.ndim == 2:
        lead = a.shape[:-1]
        out = _mm2(a.reshape(-1, a.shape[-1]), b)
        return out.reshape(lead + (b.shape[1],))
    # batched right operand: broadcast the batch dims, one GEMM per matrix
    shape = np.broadcast_shapes(a.shape[:-2], b.shape[:-2])
    ab = np.broadcast_to(a, shape + a.shape[-2:])
    bb = np.broadcast_to(b, shape + b.shape[-2:])
    out = np.empty(shape + (a.shape[-2], b.shape[-1]), np.float32)
    for idx in np.ndindex(*shape):
        out[idx] = _mm2(ab[idx], bb[idx])
    return out


def _binary(op: int, a, b) -> np.ndarray:
    a, b = np.broadcast_arrays(np.asarray(a, np.float32), np.asarray(b, np.float32))
    a, b = _f32(a), _f32(b)
    out = np.empty(a.shape, np.float32)
    if a.size:
        check(lib.rvc_cuda_elementwise(_ctx(), op, fptr(a), fptr(b), a.size, 0.0, fptr(out)))
    return out


def _unary(op: int, a, alpha: float = 0.0) -> np.ndarray:
    a = _f32(a)
    out = np.empty(a.shape, np.float32)
    if a.size:
        check(lib.rvc_cuda_elementwise(_ctx(), op, fptr(a), None, a.size, float(alpha), fptr(out)))
    return out


def add(a, b):
    """``a + b`` with numpy broadcasting (``runtime/backend.py:212-216``)."""
    return _binary(0, a, b)


def mul(a, b):
    """``a * b`` (``runtime/backend.py:219-223``)."""
    return _binary(1, a, b)


def add_inplace(a, b, buf_a=None, buf_b=None):
    """Same value as ``a + b`` (``runtime/backend.py:270-274``)."""
    return _binary(0, a, b)


def mul_inplace(a, b, buf_a=None, buf_b=None):
    """Same value as ``a * b`` (``runtime/backend.py:277-281``)."""
    return _binary(1, a, b)


def relu(a):
    """``maximum(a, 0)`` (``runtime/backend.py:226-230``)."""
    return _unary(2, a)


def leaky_relu(x, negative_slope=0.1):
    """``x if x >= 0 else slope*x`` (``runtime/nn.py:507-517``)."""
    return _unary(3, x, negative_slope)


def gelu(x):
    """Exact-erf GELU (``runtime/models/hubert.py:229-244``)."""
    return _unary(4, x)


def _pads(padding):
    if isinstance(padding, (tuple, list)):
        return int(padding[0]), int(padding[1])
    return int(padding), int(padding)


def conv1d(x, w, b=None, stride=1, padding=0, dilation=1, buf_w=None, buf_b=None):
    """torch-semantics conv1d on ``[B,C,T]`` (``runtime/backend.py:233-239``,
    numpy reference ``runtime/nn.py:90-135``)."""
    x = _f32(x)
    w = _f32(w)
    if x.ndim != 3 or w.ndim != 3 or x.shape[1] != w.shape[1]:
        raise ValueError(f"conv1d: x {x.shape} / w {w.shape} mismatch")
    pl, pr = _pads(padding)
    B, Cc, T = x.shape
    O, _, K = w.shape
    stride, dilation = int(stride), int(dilation)
    oL = (T + pl + pr - dilation * (K - 1) - 1) // stride + 1
    if oL <= 0:
        return np.zeros((B, O, 0), np.float32)
    out = np.empty((B, O, oL), np.float32)
    bb = _f32(b) if b is not None else None
    check(lib.rvc_cuda_conv1d(_ctx(), fptr(x), B, Cc, T, fptr(w), O, K, fptr(bb) if bb is not None else None,
                              stride, pl, pr, dilation, fptr(out), oL))
    return out


def conv_transpose1d(x, w, b=None, stride=1, padding=0, output_padding=0, dilation=1, buf_w=None, buf_b=None):
    """torch-semantics transposed conv1d, ``w [C_in, C_out, K]``
    (``runtime/backend.py:242-251``, numpy reference ``runtime/nn.py:294-346``)."""
    x = _f32(x)
    w = _f32(w)
    if x.ndim != 3 or w.ndim != 3 or x.shape[1] != w.shape[0]:
        raise ValueError(f"conv_transpose1d: x {x.shape} / w {w.shape} mismatch")
    B, Ci, T = x.shape
    _, Co, K = w.shape
    stride, padding = int(stride), int(padding)
    oL = (T - 1) * stride - 2 * padding + int(dilation) * (K - 1) + int(output_padding) + 1
    if oL <= 0:
        return np.zeros((B, Co, 0), np.float32)
    out = np.empty((B, Co, oL), np.float32)
    bb = _f32(b) if b is not None else None
    check(lib.rvc_cuda_conv_transpose1d(_ctx(), fptr(x), B, Ci, T, fptr(w), Co, K,
                                        fptr(bb) if bb is not None else None, stride, padding,
                                        int(output_padding), int(dilation), fptr(out), oL))
    return out


def embedding(ids, table, buf_table=None):
    """Row gather, negative ids count from the end (``runtime/nn.py:574-594``)."""
    ids = np.asarray(ids)
    table = np.asarray(table)
    if not np.issubdtype(ids.dtype, np.integer) or table.ndim != 2:
        raise TypeError("embedding: integer ids and a 2-D table are required")
    t = _f32(table)
    V, E = t.shape
    flat = np.ascontiguousarray(ids.reshape(-1), dtype=np.int64)
    if flat.size and (flat.min() < -V or flat.max() >= V):
        raise ValueError("embedding: id out of range")
    out = np.empty((flat.size, E), np.float32)
    if flat.size:
        check(lib.rvc_cuda_embedding(_ctx(), iptr(flat), flat.size, fptr(t), V, E, fptr(out)))
    return out.reshape(ids.shape + (E,))


def layer_norm(x, gamma, beta, eps=1e-5, buf_gamma=None, buf_beta=None):
    """LayerNorm over the last axis, biased variance (``runtime/backend.py:286-296``)."""
    x = _f32(x)
    C = x.shape[-1]
    out = np.empty(x.shape, np.float32)
    rows = x.size // C if C else 0
    if rows:
        check(lib.rvc_cuda_layer_norm(_ctx(), fptr(x), rows, C, fptr(_f32(gamma)), fptr(_f32(beta)),
                                      float(eps), fptr(out)))
    return out


def rmsnorm(x, gamma, eps=1e-5, buf_gamma=None):
    """RMSNorm over the last axis: ``x / sqrt(mean(x^2) + eps) * gamma``
    (``runtime/backend.py:309-316``)."""
    x = _f32(x)
    C = x.shape[-1]
    out = np.empty(x.shape, np.float32)
    rows = x.size // C if C else 0
    if rows:
        check(lib.rvc_cuda_rmsnorm(_ctx(), fptr(x), rows, C, fptr(_f32(gamma)), float(eps), fptr(out)))
    return out


def _pair(v, name):
    if isinstance(v, (tuple, list)):
        if len(v) != 2:
            raise ValueError(f"conv2d: {name} must be an int or a pair, got {v!r}")
        return int(v[0]), int(v[1])
    return int(v), int(v)


def conv2d(x, w, b=None, stride=1, padding=0, buf_w=None, buf_b=None):
    """2-D convolution with ``torch.nn.functional.conv2d`` semantics (symmetric
    zero padding), ``runtime/backend.py:254-260`` / ``runtime/nn.py:259-290``:
    ``x [B,C,H,W]``, ``w [O,C,KH,KW]``, ``b [O]`` or None -> ``[B,O,Ho,Wo]``.
    Shape errors raise ``ValueError`` (the caller then takes its numpy path)."""
    x, w = _f32(x), _f32(w)
    if x.ndim != 4 or w.ndim != 4 or x.shape[1] != w.shape[1]:
        raise ValueError(f"conv2d: x {x.shape} and w {w.shape} do not match [B,C,H,W] / [O,C,KH,KW]")
    sh, sw = _pair(stride, "stride")
    ph, pw = _pair(padding, "padding")
    B, C, H, W = x.shape
    O, _, KH, KW = w.shape
    if sh < 1 or sw < 1 or ph < 0 or pw < 0 or H + 2 * ph < KH or W + 2 * pw < KW:
        raise ValueError("conv2d: bad stride / padding for these shapes")
    Ho, Wo = (H + 2 * ph - KH) // sh + 1, (W + 2 * pw - KW) // sw + 1
    bb = None if b is None else _f32(b).reshape(-1)
    if bb is not None and bb.size != O:
        raise ValueError(f"conv2d: bias of {bb.size} values for {O} output channels")
    out = np.empty((B, O, Ho, Wo), np.float32)
    if B:
        check(lib.rvc_cuda_conv2d(_ctx(), fptr(x), B, C, H, W, fptr(w), O, KH, KW,
                                  fptr(bb) if bb is not None else None, sh, sw, ph, pw, fptr(out)))
    return out


def softmax(x):
    """Row softmax over the last axis (``runtime/backend.py:298-306``)."""
    x = _f32(x)
    C = x.shape[-1]
    out = np.empty(x.shape, np.float32)
    rows = x.size // C if C else 0
    if rows:
        check(lib.rvc_cuda_softmax(_ctx(), fptr(x), rows, C, fptr(out)))
    return out


def gating(x, g=None):
    """WaveNet gate ``tanh(x[:, :H] + g[:, :H]) * sigmoid(x[:, H:] + g[:, H:])``
    on ``x [B, 2H, T]``, ``g [B, 2H, 1]`` (``runtime/models/vits.py:1131-1132``)."""
    x = _f32(x)
    B, H2, T = x.shape
    H = H2 // 2
    out = np.empty((B, H, T), np.float32)
    gg = _f32(np.broadcast_to(np.asarray(g, np.float32), (B, H2, 1))) if g is not None else None
    check(lib.rvc_cuda_gating(_ctx(), fptr(x), fptr(gg) if gg is not None else None, B, H, T, fptr(out)))
    return out


def rel_attention(q, k, v, emb_rel_k, emb_rel_v, heads, window=10):
    """Text-encoder attention with T5 relative positions for one layer.

    ``q, k, v [B, heads*kc, P]`` (projected), ``emb_rel_k/v [1, 2*window+1, kc]``
    -> ``[B, heads*kc, P]``; ``runtime/models/vits.py:993-1014``.
    """
    q, k, v = _f32(q), _f32(k), _f32(v)
    B, Hc, P = q.shape
    kc = Hc // int(heads)
    ek = _f32(np.asarray(emb_rel_k).reshape(-1, kc))
    ev = _f32(np.asarray(emb_rel_v).reshape(-1, kc))
    out = np.empty((B, Hc, P), np.float32)
    check(lib.rvc_cuda_rel_attention(_ctx(), fptr(q), fptr(k), fptr(v), fptr(ek), fptr(ev), B, int(heads), kc, P,
                                     int(window), fptr(out)))
    return out


def im2col_1d(x, kernel_size, stride=1, padding=0, dilation=1):
    """``x [B,C,T]`` -> ``cols [B, oL, C*K]`` (column c*K+k), the layout of the
    reference engine's im2col_1d (``runtime/vulkan_ops.py:2727``)."""
    x = _f32(x)
    B, Cc, T = x.shape
    pl, pr = _pads(padding)
    K = int(kernel_size)
    oL = (T + pl + pr - int(dilation) * (K - 1) - 1) // int(stride) + 1
    out = np.empty((B, max(oL, 0), Cc * K), np.float32)
    if oL > 0:
        check(lib.rvc_cuda_im2col1d(_ctx(), fptr(x), B, Cc, T, K, int(stride), pl, int(dilation), oL, fptr(out)))
    return out


# ------------------------------------------------------- attention operators
# Host forms of rvc_cuda.attention: float32 numpy arrays in and out, on the
# default context's device and stream.  They need no torch.


class _Scratch:
    """Device memory of one call: inputs, results and workspace from the context's
    pool, given back when the call ends (the pool is reused in stream order)."""

    def __init__(self):
        self.ctx = _lib.get_context()
        self.handle, self.stream = self.ctx.handle, self.ctx.stream()
        self.held = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for p in self.held:
            self.ctx.free(p)

    def new(self, nbytes: int) -> int:
        p = self.ctx.alloc(max(16, nbytes))
        self.held.append(p)
        return p

    def up(self, a):
        """Device copy of an array (None stays None)."""
        if a is None:
            return None
        p = self.new(a.nbytes)
        if a.nbytes:
            self.ctx.h2d(p, a)
        return p

    def out(self, *shapes):
        return [self.new(4 * int(np.prod(s))) for s in shapes]

    def workspace(self, fn, desc, n, *how):
        need = C.c_int64(0)
        check(fn(self.handle, desc, n, *how, need))
        return (self.new(need.value) if need.value else None), need.value

    def down(self, p: int, shape) -> np.ndarray:
        a = np.empty(shape, np.float32)
        if a.nbytes:
            self.ctx.d2h(a, p)
        return a


def _dims(a, name: str, ndim: int) -> np.ndarray:
    a = _f32(a)
    if a.ndim != ndim:
        raise ValueError(f"{name}: {ndim} dimensions expected, got shape {a.shape}")
    return a


def _whole(a, name: str) -> np.ndarray:
    a = np.asarray(a)
    if not np.issubdtype(a.dtype, np.integer):
        raise ValueError(f"{name}: integers are expected")
    return np.ascontiguousarray(a, dtype=np.int64)


def _rows(a) -> tuple:
    """Strides (batch, row, head) of a contiguous [B, L, H, D]."""
    _, L, H, D = a.shape
    return L * H * D, H * D, D


def _host_bias(bias):
    if not isinstance(bias, BucketBias):
        raise ValueError("bias: an rvc_cuda.attention.BucketBias is expected")
    t = _dims(bias.table, "bias table", 2)
    if t.shape[0] != bias.num_buckets:
        raise ValueError(f"bias: table {t.shape}, its rows must be the {bias.num_buckets} buckets")
    return t


def _host_attention(q, k, v, kv_lens, key_mask, scale, causal, q_offset, bias, rest=()):
    """(q, k, v, lens, mask, table, descriptor, scale, borders and their count); ``rest``: dout and out."""
    q, k, v = _dims(q, "q", 4), _dims(k, "k", 4), _dims(v, "v", 4)
    B, Lq, Hq, D = q.shape
    Bk, Lk, Hkv, Dk = k.shape
    if Bk != B or Dk != D or v.shape != k.shape:
        raise ValueError(f"attention: q {q.shape}, k {k.shape}, v {v.shape} do not match [B, Lq, Hq, D] and [B, Lk, Hkv, D]")
    if not 1 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"attention: head dimension {D}; 1 to {MAX_HEAD_DIM} are supported")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"attention: {Hq} query heads are no multiple of {Hkv} key heads")
    lens = mask = table = None
    if kv_lens is not None:
        lens = _whole(kv_lens, "kv_lens")
        if lens.shape != (B,):
            raise ValueError(f"kv_lens: [{B}] expected, got {lens.shape}")
    if key_mask is not None:
        mask = np.ascontiguousarray(key_mask, dtype=np.bool_)
        if mask.shape != (B, Lk):
            raise ValueError(f"key_mask: [{B}, {Lk}] expected, got {mask.shape}")
    if bias is not None:
        table = _host_bias(bias)
        if table.shape[1] != Hq:
            raise ValueError(f"bias: table {table.shape}, expected [{bias.num_buckets}, {Hq}] for {Hq} query heads")
    desc = _pack29(0, B, Hq, Hkv, Lq, Lk, D, *_rows(q), *_rows(k), *_rows(v), 64 if lens is not None else 0,
                   Lk if mask is not None else 0, 1 if mask is not None else 0, bool(causal), _offset(q_offset),
                   bias.num_buckets if bias is not None else 0, bias.bidirectional if bias is not None else 0,
                   *(_rows(q) * 2 if rest else (0,) * 6))
    borders, n = (bias._borders, bias._nborders) if bias is not None else (None, 0)
    return q, k, v, lens, mask, table, desc, _scale(scale, D), borders, n


def attention(q, k, v, kv_lens=None, key_mask=None, scale=None, causal=False, q_offset=0, bias=None):
    """``rvc_cuda.attention.attention`` for numpy arrays: ``q [B, Lq, Hq, D]``,
    ``k, v [B, Lk, Hkv, D]`` -> ``(out, lse)``; the table of ``bias`` (a
    ``BucketBias``) is a numpy array too."""
    q, k, v, lens, mask, table, desc, scale, borders, n = _host_attention(q, k, v, kv_lens, key_mask, scale, causal,
                                                                          q_offset, bias)
    B, Lq, Hq, _ = q.shape
    with _Scratch() as d:
        out, lse = d.out(q.shape, (B, Hq, Lq))
        ws, nbytes = d.workspace(lib.rvc_cuda_attention_workspace, desc, 29, 0)
        check(lib.rvc_cuda_attention_device(d.handle, d.stream, desc, 29, scale, d.up(q), d.up(k), d.up(v), d.up(lens),
                                            d.up(mask), d.up(table), borders, n, out, lse, ws, nbytes))
        return d.down(out, q.shape), d.down(lse, (B, Hq, Lq))


def attention_backward(dout, q, k, v, out, lse, kv_lens=None, key_mask=None, scale=None, causal=False, q_offset=0,
                       bias=None):
    """``rvc_cuda.attention.attention_backward`` for numpy arrays."""
    q, k, v, lens, mask, table, desc, scale, borders, n = _host_attention(q, k, v, kv_lens, key_mask, scale, causal,
                                                                          q_offset, bias, (dout, out))
    dout, out, lse = _dims(dout, "dout", 4), _dims(out, "out", 4), _dims(lse, "lse", 3)
    B, Lq, Hq, _ = q.shape
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"attention_backward: dout {dout.shape} and out {out.shape} must have the shape of q {q.shape}")
    if lse.shape != (B, Hq, Lq):
        raise ValueError(f"attention_backward: lse must be [{B}, {Hq}, {Lq}], got {lse.shape}")
    with _Scratch() as d:
        shapes = [q.shape, k.shape, v.shape] + ([table.shape] if table is not None else [])
        grads = d.out(*shapes)
        ws, nbytes = d.workspace(lib.rvc_cuda_attention_workspace, desc, 29, 1)
        check(lib.rvc_cuda_attention_backward_device(
            d.handle, d.stream, desc, 29, scale, d.up(dout), d.up(q), d.up(k), d.up(v), d.up(out), d.up(lse), d.up(lens),
            d.up(mask), d.up(table), borders, n, *grads[:3], grads[3] if table is not None else None, ws, nbytes))
        return tuple(d.down(p, s) for p, s in zip(grads, shapes))


def relative_bias(bias, Lq, Lk, q_offset=0):
    """``rvc_cuda.attention.relative_bias`` with a numpy table -> ``[heads, Lq, Lk]``."""
    table = _host_bias(bias)
    shape = (table.shape[1], _length(Lq), _length(Lk))
    desc = _pack11(0, 1, *shape, _offset(q_offset), bias.num_buckets, bias.bidirectional, 0, 0, 0)
    with _Scratch() as d:
        out, = d.out(shape)
        check(lib.rvc_cuda_relative_bias_device(d.handle, d.stream, desc, 11, d.up(table), bias._borders, bias._nborders,
                                                out))
        return d.down(out, shape)


def relative_bias_backward(bias, dbias, q_offset=0):
    """``rvc_cuda.attention.relative_bias_backward`` for numpy arrays."""
    table, dbias = _host_bias(bias), _f32(dbias)
    dbias = _dims(dbias[None] if dbias.ndim == 3 else dbias, "dbias", 4)
    B, H, Lq, Lk = dbias.shape
    if H != table.shape[1]:
        raise ValueError(f"relative_bias_backward: {H} heads, the table has {table.shape[1]}")
    desc = _pack11(0, B, H, Lq, Lk, _offset(q_offset), bias.num_buckets, bias.bidirectional, H * Lq * Lk, Lq * Lk, Lk)
    with _Scratch() as d:
        out, = d.out(table.shape)
        ws, nbytes = d.workspace(lib.rvc_cuda_relative_bias_workspace, desc, 11)
        check(lib.rvc_cuda_relative_bias_backward_device(d.handle, d.stream, desc, 11, d.up(dbias), bias._borders,
                                                         bias._nborders, out, ws, nbytes))
        return d.down(out, table.shape)


def _host_rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved, name, grads=()):
    """The arrays, and the descriptor."""
    q, k = _dims(q, "q", 4), _dims(k, "k", 4)
    wq, wk, cos, sin = _dims(q_weight, "q_weight", 1), _dims(k_weight, "k_weight", 1), _dims(cos, "cos", 2), _dims(sin, "sin", 2)
    B, L, Hq, D = q.shape
    if k.shape[:2] != (B, L) or k.shape[3] != D:
        raise ValueError(f"{name}: q {q.shape} and k {k.shape} do not match [B, L, heads, D]")
    if D < 2 or D > 256 or D % 2:
        raise ValueError(f"{name}: head dimension {D}; even ones from 2 to 256 are supported")
    if wq.shape != (D,) or wk.shape != (D,):
        raise ValueError(f"{name}: weights [{D}] expected, got {wq.shape} and {wk.shape}")
    if cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise ValueError(f"{name}: cos {cos.shape} and sin {sin.shape} do not fit head dimension {D}")
    bits = pb = pl = 0
    pos = None
    if positions is not None:
        pos = _whole(positions, "positions")
        if pos.shape == (B, L):
            pb, pl = L, 1
        elif pos.shape == (L,):
            pl = 1
        else:
            raise ValueError(f"{name}: positions [{B}, {L}] or [{L}] expected, got {pos.shape}")
        bits = 64
    elif L > cos.shape[0] and cos.shape[1]:
        raise ValueError(f"{name}: the tables hold {cos.shape[0]} positions, fewer than the {L} rows")
    grads = [_dims(g, n, 4) for g, n in zip(grads, ("dqo", "dko"))]
    for g, x in zip(grads, (q, k)):
        if g.shape != x.shape:
            raise ValueError(f"{name}: a gradient {g.shape} for {x.shape}")
    desc = _pack25(0, 0, B, L, Hq, k.shape[2], D, 2 * cos.shape[1], cos.shape[0], bool(interleaved), bits, pb, pl,
                   *_rows(q), *_rows(k), *(_rows(q) + _rows(k) if grads else (0,) * 6))
    return [*grads, q, k, wq, wk, cos, sin, pos], desc


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False):
    """``rvc_cuda.attention.qk_norm_rope`` for numpy arrays."""
    arrays, desc = _host_rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved, "qk_norm_rope")
    shapes = [a.shape for a in arrays[:2]]
    with _Scratch() as d:
        out = d.out(*shapes)
        check(lib.rvc_cuda_qk_norm_rope_device(d.handle, d.stream, desc, 25, float(eps), *map(d.up, arrays), *out))
        return tuple(d.down(p, s) for p, s in zip(out, shapes))


def qk_norm_rope_backward(dqo, dko, q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False):
    """``rvc_cuda.attention.qk_norm_rope_backward`` for numpy arrays."""
    arrays, desc = _host_rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved, "qk_norm_rope_backward",
                              (dqo, dko))
    shapes = [a.shape for a in arrays[2:6]]
    with _Scratch() as d:
        out = d.out(*shapes)
        ws, nbytes = d.workspace(lib.rvc_cuda_qk_norm_rope_workspace, desc, 25)
        check(lib.rvc_cuda_qk_norm_rope_backward_device(d.handle, d.stream, desc, 25, float(eps), *map(d.up, arrays), *out,
                                                        ws, nbytes))
        r = [d.down(p, s) for p, s in zip(out, shapes)]
    if arrays[3].shape[2] == 0:  # no keys: nobody writes their weight's gradient
        r[3][:] = 0
    return tuple(r)
