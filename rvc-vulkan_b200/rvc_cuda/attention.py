"""Attention operators on device tensors, with their gradients.

* ``attention`` / ``attention_backward``: softmax attention of queries over
  keys and values of another length (an encoder's states, a cache) or their
  own, with padded batches, shared key/value heads, a causal limit and a
  learned bias of the distance;
* ``relative_bias`` / ``relative_bias_backward``: that bias as a tensor, and
  the gradient of its table from a gradient of the tensor;
* ``qk_norm_rope`` / ``qk_norm_rope_backward``: the RMS norm of every query and
  key head with the rotation of its position, in one pass.

The functions take CUDA tensors (``torch.float32``, ``bfloat16`` or
``float16``), run on the tensors' device and its current stream without
synchronising, and return new contiguous tensors; scratch memory comes from
torch's allocator, so a call can be captured into a CUDA graph (after a first
call on the device, which opens the library's context there).  Nothing is kept
between calls, and there is no autograd: the ``*_backward`` functions are called
with what the forward ones returned, and an input that requires grad is refused
while grad mode is on (call under ``torch.no_grad()`` or inside an
``autograd.Function``, where it is off).  A wait inside a kernel that gives up
(after two seconds) leaves NaN in the results that waited and is reported by the
next ``sync`` of the device's context, ``rvc_cuda._lib.get_context(i).sync()``.
``rvc_cuda.ops`` has the forms for numpy arrays.  The device code and its C entry
points (``include/rvc_cuda.h``) have no counterpart in the reference, whose
attention (``runtime/models/vits.py:993-1014``,
``runtime/models/hubert.py:1315-1400``) has one length, no padding and no
gradient.  A shape, type or argument that is not served raises ``ValueError``.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._attn_args import (MAX_BUCKETS, MAX_HEAD_DIM, MAX_SCALE, BucketBias, _length, _offset,  # noqa: F401
                         _pack11, _pack25, _pack29, _scale, bucket_borders)
from ._lib import check, lib

__all__ = ["BucketBias", "attention", "attention_backward", "relative_bias", "relative_bias_backward",
           "qk_norm_rope", "qk_norm_rope_backward", "rope_table"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# torch's own short way to the current stream's handle, a microsecond less than the public one
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda i: torch.cuda.current_stream(i).cuda_stream)
_POSITION_BITS = {torch.int32: 32, torch.int64: 64}


# ------------------------------------------------------------------ plumbing


def _tensor(x, name: str, ndim: int, like=None):
    """``x`` with its last dimension contiguous, checked against ``like``."""
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name}: a tensor is expected")
    if x.dim() != ndim:
        raise ValueError(f"{name}: {ndim} dimensions expected, got shape {tuple(x.shape)}")
    if like is None:
        if x.dtype not in _TYPES:
            raise ValueError(f"{name}: float32, bfloat16 or float16 expected, got {x.dtype}")
    elif x.dtype is not like.dtype:
        raise ValueError(f"{name}: {like.dtype} expected, got {x.dtype}")
    elif x.get_device() != like.get_device():
        raise ValueError(f"{name}: on {x.device}, expected {like.device}")
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _where(x):
    """(context handle, raw stream of the tensor's device)."""
    i = x.get_device()
    if i < 0:
        raise ValueError(f"CUDA tensors are expected, got one on {x.device}")
    return _lib.get_context(i).handle, _raw_stream(i)


def _scratch(fn, ctx, desc, n, like, *how):
    """Workspace that ``fn`` (a ``*_workspace`` entry) asks for: (tensor or None, bytes)."""
    need = C.c_int64(0)
    check(fn(ctx, desc, n, *how, need))
    nbytes = need.value
    return (like.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None), nbytes


def _no_graph(name: str, *tensors):
    """Results have no graph behind them: a gradient that autograd was asked for would be lost without a word."""
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                raise ValueError(f"{name}: an input requires grad, and this function records no graph: call it under "
                                 "torch.no_grad() and use the *_backward functions")


def _ptr(x):
    return x.data_ptr() if x is not None else None


def _qkv(q, k, v):
    try:  # the ordinary call in few steps; what is not ordinary is looked at one by one below
        B, Lq, Hq, D = q.shape
        Bk, Lk, Hkv, Dk = k.shape
        t, i = q.dtype, q.get_device()
        if (Bk == B and Dk == D and v.shape == k.shape and k.dtype is t and v.dtype is t and t in _TYPES
                and k.get_device() == i and v.get_device() == i and 1 <= D <= MAX_HEAD_DIM and Hkv and Hq
                and Hq % Hkv == 0 and q.stride(3) == 1 and k.stride(3) == 1 and v.stride(3) == 1):
            return q, k, v, B, Lq, Lk, Hq, Hkv, D
    except (AttributeError, ValueError):
        pass
    q = _tensor(q, "q", 4)
    k, v = _tensor(k, "k", 4, q), _tensor(v, "v", 4, q)
    B, Lq, Hq, D = q.shape
    Bk, Lk, Hkv, Dk = k.shape
    if Bk != B or Dk != D or v.shape != k.shape:
        raise ValueError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match "
                         "[B, Lq, Hq, D] and [B, Lk, Hkv, D]")
    if not 1 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"attention: head dimension {D}; 1 to {MAX_HEAD_DIM} are supported")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"attention: {Hq} query heads are no multiple of {Hkv} key heads")
    return q, k, v, B, Lq, Lk, Hq, Hkv, D


def _lens(kv_lens, B: int, like):
    if kv_lens is None:
        return None, 0
    if not isinstance(kv_lens, torch.Tensor) or kv_lens.device != like.device:
        raise ValueError(f"kv_lens: a tensor on {like.device} is expected")
    if kv_lens.shape != (B,) or kv_lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"kv_lens: int32 or int64 [{B}] expected, got {kv_lens.dtype} {tuple(kv_lens.shape)}")
    return kv_lens.contiguous(), 32 if kv_lens.dtype == torch.int32 else 64


def _mask(key_mask, B: int, Lk: int, like):
    if key_mask is None:
        return None, 0, 0
    if not isinstance(key_mask, torch.Tensor) or key_mask.device != like.device:
        raise ValueError(f"key_mask: a tensor on {like.device} is expected")
    if key_mask.shape != (B, Lk) or key_mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"key_mask: bool or uint8 [{B}, {Lk}] expected, got {key_mask.dtype} {tuple(key_mask.shape)}")
    return key_mask, key_mask.stride(0), key_mask.stride(1)


def _rows(bias, t):
    """The object's table ``t`` (which may have been replaced) has the rows that its borders lead to."""
    if t.shape[0] != bias.num_buckets:
        raise ValueError(f"bias: table {tuple(t.shape)}, its rows must be the {bias.num_buckets} buckets")


def _table(bias, H: int, like):
    """The table as the kernels read it (contiguous), its size and borders."""
    if bias is None:
        return None, 0, 0, None, 0
    if not isinstance(bias, BucketBias):
        raise ValueError("bias: a BucketBias is expected")
    t = _tensor(bias.table, "bias table", 2, like)
    _rows(bias, t)
    if t.shape[1] != H:
        raise ValueError(f"bias: table {tuple(t.shape)}, expected [{bias.num_buckets}, {H}] for {H} query heads")
    return t.contiguous(), bias.num_buckets, int(bias.bidirectional), bias._borders, bias._nborders


# ----------------------------------------------------------------- attention


def attention(q, k, v, *, kv_lens=None, key_mask=None, scale: Optional[float] = None, causal: bool = False,
              q_offset: int = 0, bias: Optional[BucketBias] = None):
    """Attention of ``q [B, Lq, Hq, D]`` over ``k, v [B, Lk, Hkv, D]``.

    ``softmax(scale q k^T + bias) v`` over the live keys of each batch entry:
    those before ``kv_lens [B]`` (int32 or int64, clamped to ``[0, Lk]``), with
    ``key_mask [B, Lk]`` (bool or uint8) set, and, when ``causal``, not past
    ``i + q_offset`` for query ``i`` (``q_offset = Lk - Lq`` aligns the last
    query with the last key).  Whatever a key holds that no query meets reaches
    no result: padding, masked keys, a cache past the last query's limit.  A key
    that is past the limit of some queries only, or masked by the bias alone, must
    be finite, as its weight of 0 there meets the value.
    Query head ``h`` reads key head ``h // (Hq / Hkv)``.  ``scale`` is
    ``1 / sqrt(D)`` by default; ``bias`` adds ``table[bucket(j - i - q_offset),
    h]`` (an entry below -65536 masks its pairs: ``-inf``, ``-1e9``, the lowest
    float32 and bfloat16).  Other entries and scores are meant to stay below 1e5
    in size, as gradients take their weights from the float32 log sums.  Returns ``out [B, Lq, Hq, D]`` in the type of ``q`` and the float32
    log sums ``lse [B, Hq, Lq]`` that the backward pass takes; a query without
    a live key gives 0 and ``-inf``.  float32 values are worked on as parts of
    16 bits: an infinite one that is alive comes out as NaN.  Heads of 1 to 128
    values; any strides
    (the parts of a packed projection are taken where they lie).
    """
    q, k, v, B, Lq, Lk, Hq, Hkv, D = _qkv(q, k, v)
    lens = mask = table = borders = None
    bits = mb = mk = nb = both = nborders = 0
    if kv_lens is not None:
        lens, bits = _lens(kv_lens, B, q)
    if key_mask is not None:
        mask, mb, mk = _mask(key_mask, B, Lk, q)
    if bias is not None:
        table, nb, both, borders, nborders = _table(bias, Hq, q)
    _no_graph("attention", q, k, v, table)
    ctx, stream = _where(q)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    desc = _pack29(_TYPES[q.dtype], B, Hq, Hkv, Lq, Lk, D, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1],
                   vs[2], bits, mb, mk, bool(causal), _offset(q_offset), nb, both, 0, 0, 0, 0, 0, 0)
    scale = _scale(scale, D)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, Hq, Lq), dtype=torch.float32)
    ws, nbytes = _scratch(lib.rvc_cuda_attention_workspace, ctx, desc, 29, q, 0)
    check(lib.rvc_cuda_attention_device(ctx, stream, desc, 29, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                        _ptr(lens), _ptr(mask), _ptr(table), borders, nborders, out.data_ptr(),
                                        lse.data_ptr(), _ptr(ws), nbytes))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, kv_lens=None, key_mask=None, scale: Optional[float] = None,
                       causal: bool = False, q_offset: int = 0, bias: Optional[BucketBias] = None):
    """Gradients of ``attention`` for ``dout [B, Lq, Hq, D]``.

    ``out`` and ``lse`` are what ``attention`` returned for the same arguments.
    Returns ``(dq, dk, dv)``, and ``dtable [num_buckets, Hq]`` behind them when
    a ``bias`` is given, in the types of their inputs; a key head's gradient is
    the sum over the query heads that share it.  Dead keys and queries without
    a live key get zeros, and so do ``q``, ``k`` and the table from a query that
    length, mask and causal limit leave one key.  Sums run in a fixed order: the
    same call gives the same bits.  With a ``bias`` the scratch memory grows with
    ``Lq Lk``, up to ``B Hq Lq Lk / 16`` bytes.  float16 gradients want a loss
    scale that keeps ``p (dout v - sum p dout v)``, which is rounded to float16 on
    the way, between its subnormals and 65504.
    """
    q, k, v, B, Lq, Lk, Hq, Hkv, D = _qkv(q, k, v)
    dout, out = _tensor(dout, "dout", 4, q), _tensor(out, "out", 4, q)
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"attention_backward: dout {tuple(dout.shape)} and out {tuple(out.shape)} must have the shape "
                         f"of q {tuple(q.shape)}")
    if (not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.shape != (B, Hq, Lq)
            or lse.device != q.device):
        raise ValueError(f"attention_backward: lse must be float32 [{B}, {Hq}, {Lq}] on {q.device}")
    lse = lse.contiguous()
    lens, bits = _lens(kv_lens, B, q)
    mask, mb, mk = _mask(key_mask, B, Lk, q)
    table, nb, both, borders, nborders = _table(bias, Hq, q)
    _no_graph("attention_backward", dout, q, k, v, out, lse, table)
    ctx, stream = _where(q)
    desc = _pack29(_TYPES[q.dtype], B, Hq, Hkv, Lq, Lk, D, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], bits, mb,
                   mk, bool(causal), _offset(q_offset), nb, both, *dout.stride()[:3], *out.stride()[:3])
    dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    dtable = q.new_empty((nb, Hq)) if nb else None
    ws, nbytes = _scratch(lib.rvc_cuda_attention_workspace, ctx, desc, 29, q, 1)
    check(lib.rvc_cuda_attention_backward_device(
        ctx, stream, desc, 29, _scale(scale, D), dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
        out.data_ptr(), lse.data_ptr(), _ptr(lens), _ptr(mask), _ptr(table), borders, nborders, dq.data_ptr(),
        dk.data_ptr(), dv.data_ptr(), _ptr(dtable), _ptr(ws), nbytes))
    return (dq, dk, dv) if dtable is None else (dq, dk, dv, dtable)


# ------------------------------------------------------------- bias of distance


def relative_bias(bias: BucketBias, Lq: int, Lk: int, *, q_offset: int = 0):
    """The bias as a tensor: ``[heads, Lq, Lk]`` in the table's type, entry
    ``(h, i, j)`` is ``table[bucket(j - i - q_offset), h]``."""
    if not isinstance(bias, BucketBias):
        raise ValueError("relative_bias: a BucketBias is expected")
    t = _tensor(bias.table, "bias table", 2).contiguous()
    _rows(bias, t)
    Lq, Lk, H = _length(Lq), _length(Lk), t.shape[1]
    _no_graph("relative_bias", t)
    ctx, stream = _where(t)
    out = t.new_empty((H, Lq, Lk))
    desc = _pack11(_TYPES[t.dtype], 1, H, Lq, Lk, _offset(q_offset), bias.num_buckets, bias.bidirectional, 0, 0, 0)
    check(lib.rvc_cuda_relative_bias_device(ctx, stream, desc, 11, t.data_ptr(), bias._borders, bias._nborders,
                                            out.data_ptr()))
    return out


def relative_bias_backward(bias: BucketBias, dbias, *, q_offset: int = 0):
    """Gradient of the table from ``dbias [heads, Lq, Lk]``, or ``[B, heads, Lq,
    Lk]`` for a bias that was broadcast over a batch: ``[num_buckets, heads]``
    in the type of the table.  Sums are held in 32 bits along a diagonal's part
    and in 64 bits beyond, in a fixed order."""
    if not isinstance(bias, BucketBias):
        raise ValueError("relative_bias_backward: a BucketBias is expected")
    if isinstance(dbias, torch.Tensor) and dbias.dim() == 3:
        dbias = dbias[None]
    d = _tensor(dbias, "dbias", 4, bias.table)
    if d.dtype not in _TYPES:
        raise ValueError(f"dbias: float32, bfloat16 or float16 expected, got {d.dtype}")
    B, H, Lq, Lk = d.shape
    _rows(bias, _tensor(bias.table, "bias table", 2))
    if H != bias.table.shape[1]:
        raise ValueError(f"relative_bias_backward: {H} heads, the table has {bias.table.shape[1]}")
    _no_graph("relative_bias_backward", d)
    ctx, stream = _where(d)
    desc = _pack11(_TYPES[d.dtype], B, H, Lq, Lk, _offset(q_offset), bias.num_buckets, bias.bidirectional, *d.stride()[:3])
    dtable = d.new_empty((bias.num_buckets, H))
    ws, nbytes = _scratch(lib.rvc_cuda_relative_bias_workspace, ctx, desc, 11, d)
    check(lib.rvc_cuda_relative_bias_backward_device(ctx, stream, desc, 11, d.data_ptr(), bias._borders,
                                                     bias._nborders, dtable.data_ptr(), _ptr(ws), nbytes))
    return dtable


# ---------------------------------------------------------- norm and rotation


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None):
    """Cosines and sines ``[max_positions, rotary_dim / 2]`` (float32) of the
    angles ``position * base^(-2 i / rotary_dim)``, formed in 64 bits."""
    if rotary_dim < 2 or rotary_dim % 2 or max_positions < 1:
        raise ValueError(f"rope_table: {max_positions} positions, rotary dimension {rotary_dim}")
    f = float(base) ** (-np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim)
    a = np.arange(max_positions, dtype=np.float64)[:, None] * f
    device = torch.device("cuda") if device is None else device
    return (torch.from_numpy(np.cos(a).astype(np.float32)).to(device),
            torch.from_numpy(np.sin(a).astype(np.float32)).to(device))


def _rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved, name):
    try:  # the ordinary call in few steps; what is not ordinary is looked at one by one below
        B, L, Hq, D = q.shape
        Bk, Lk, Hk, Dk = k.shape
        P, half = cos.shape
        t, tw, i = q.dtype, q_weight.dtype, q.get_device()
        if (Bk == B and Lk == L and Dk == D and k.dtype is t and t in _TYPES and 2 <= D <= 256 and D % 2 == 0
                and (tw is torch.float32 or tw is t) and k_weight.dtype is tw and q_weight.shape == (D,)
                and k_weight.shape == (D,) and sin.shape == cos.shape and 2 * half <= D and q_weight.is_contiguous()
                and k_weight.is_contiguous() and cos.is_contiguous() and sin.is_contiguous()
                and cos.dtype is torch.float32 and sin.dtype is torch.float32 and q.stride(3) == 1 and k.stride(3) == 1
                and k.get_device() == q_weight.get_device() == k_weight.get_device() == cos.get_device()
                == sin.get_device() == positions.get_device() == i and positions.shape == (B, L)
                and positions.dtype in _POSITION_BITS and B * L):
            return q, k, q_weight, k_weight, cos, sin, positions, (
                _TYPES[t], _TYPES[tw], B, L, Hq, Hk, D, 2 * half, P, bool(interleaved),
                _POSITION_BITS[positions.dtype], *positions.stride(), *q.stride()[:3], *k.stride()[:3])
    except (AttributeError, ValueError):
        pass
    q = _tensor(q, "q", 4)
    k = _tensor(k, "k", 4, q)
    B, L, Hq, D = q.shape
    Hk = k.shape[2]
    if k.shape[:2] != q.shape[:2] or k.shape[3] != D:
        raise ValueError(f"{name}: q {tuple(q.shape)} and k {tuple(k.shape)} do not match [B, L, heads, D]")
    if D < 2 or D > 256 or D % 2:
        raise ValueError(f"{name}: head dimension {D}; even ones from 2 to 256 are supported")
    dev = q.get_device()
    for w, n in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if not isinstance(w, torch.Tensor) or w.shape != (D,) or w.get_device() != dev:
            raise ValueError(f"{name}: {n} [{D}] on {q.device} expected")
        if w.dtype not in (torch.float32, q.dtype) or w.dtype != q_weight.dtype:
            raise ValueError(f"{name}: the weights are both float32 or both {q.dtype}")
    for t, n in ((cos, "cos"), (sin, "sin")):
        if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.dtype is not torch.float32 or t.get_device() != dev:
            raise ValueError(f"{name}: {n} must be a float32 [positions, rotary_dim / 2] on {q.device}")
    if cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise ValueError(f"{name}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} do not fit head dimension {D}")
    bits = pb = pl = 0
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.get_device() != dev:
            raise ValueError(f"{name}: positions must be a tensor on {q.device}")
        if positions.shape == (B, L):
            pb, pl = positions.stride()
        elif positions.shape == (L,):
            pl = positions.stride(0)
        else:
            raise ValueError(f"{name}: positions [{B}, {L}] or [{L}] expected, got {tuple(positions.shape)}")
        if positions.dtype not in _POSITION_BITS:
            raise ValueError(f"{name}: positions are int32 or int64, got {positions.dtype}")
        bits = _POSITION_BITS[positions.dtype]
    elif L > cos.shape[0] and cos.shape[1]:
        raise ValueError(f"{name}: the tables hold {cos.shape[0]} positions, fewer than the {L} rows")
    if B * L == 0:
        positions = None
        bits = 0
    qs, ks = q.stride(), k.stride()
    head = (_TYPES[q.dtype], _TYPES[q_weight.dtype], B, L, Hq, Hk, D, 2 * cos.shape[1], cos.shape[0], bool(interleaved),
            bits, pb, pl, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2])
    return q, k, q_weight.contiguous(), k_weight.contiguous(), cos.contiguous(), sin.contiguous(), positions, head


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, positions=None, eps: float = 1e-6, interleaved: bool = False):
    """RMS norm of each head of ``q [B, L, Hq, D]`` and ``k [B, L, Hk, D]`` with
    ``q_weight`` / ``k_weight [D]`` (float32 or the type of ``q``), then the
    rotation of its position, in one pass: ``(q', k')``, contiguous.

    ``cos``, ``sin [P, R / 2]`` (float32, ``rope_table``) rotate the first ``R``
    values of a head: pairs ``(x, x + R / 2)``, or ``(2x, 2x + 1)`` when
    ``interleaved``.  ``positions [B, L]`` or ``[L]`` (int32 or int64) are rows
    of the tables, ``0 .. L - 1`` by default; a row whose position lies outside
    them comes out as NaN.
    """
    q, k, wq, wk, cos, sin, pos, head = _rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved,
                                              "qk_norm_rope")
    _no_graph("qk_norm_rope", q, k, wq, wk, cos, sin)
    ctx, stream = _where(q)
    desc = _pack25(*head, 0, 0, 0, 0, 0, 0)
    qo, ko = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
    check(lib.rvc_cuda_qk_norm_rope_device(ctx, stream, desc, 25, float(eps), q.data_ptr(), k.data_ptr(),
                                           wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), _ptr(pos),
                                           qo.data_ptr(), ko.data_ptr()))
    return qo, ko


def qk_norm_rope_backward(dqo, dko, q, k, q_weight, k_weight, cos, sin, *, positions=None, eps: float = 1e-6,
                          interleaved: bool = False):
    """Gradients of ``qk_norm_rope`` for ``dqo``, ``dko``: ``(dq, dk, dq_weight,
    dk_weight)``, each in the type of its input; the weights' sums over the rows
    are held in 32 and 64 bits and run in a fixed order."""
    q, k, wq, wk, cos, sin, pos, head = _rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved,
                                              "qk_norm_rope_backward")
    gq, gk = _tensor(dqo, "dqo", 4, q), _tensor(dko, "dko", 4, q)
    if gq.shape != q.shape or gk.shape != k.shape:
        raise ValueError(f"qk_norm_rope_backward: dqo {tuple(gq.shape)}, dko {tuple(gk.shape)} for q {tuple(q.shape)}, "
                         f"k {tuple(k.shape)}")
    _no_graph("qk_norm_rope_backward", gq, gk, q, k, wq, wk, cos, sin)
    ctx, stream = _where(q)
    desc = _pack25(*head, *gq.stride()[:3], *gk.stride()[:3])
    dq, dk = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
    dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
    if k.shape[2] == 0:
        dwk.zero_()
    ws, nbytes = _scratch(lib.rvc_cuda_qk_norm_rope_workspace, ctx, desc, 25, q)
    check(lib.rvc_cuda_qk_norm_rope_backward_device(
        ctx, stream, desc, 25, float(eps), gq.data_ptr(), gk.data_ptr(), q.data_ptr(), k.data_ptr(), wq.data_ptr(),
        wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), _ptr(pos), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(),
        dwk.data_ptr(), _ptr(ws), nbytes))
    return dq, dk, dwq, dwk
