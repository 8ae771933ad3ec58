"""Arguments of the attention operators that are no tensors: the buckets of the
bias of distance, scale, offset, lengths, and the packed descriptors of the C
calls.  Shared by ``rvc_cuda.attention`` (torch tensors) and ``rvc_cuda.ops``
(numpy arrays, without torch)."""

from __future__ import annotations

import ctypes as C
import functools
import math
import operator
import struct

MAX_HEAD_DIM = 128
MAX_BUCKETS = 1024
MAX_SCALE = 2.0 ** 127  # times log2 e it is still a float32

_pack29 = struct.Struct("=29q").pack
_pack25 = struct.Struct("=25q").pack
_pack11 = struct.Struct("=11q").pack


@functools.lru_cache(maxsize=64)
def bucket_borders(num_buckets: int, max_distance: int, bidirectional: bool = True) -> tuple:
    """Smallest distances of the buckets 1, 2, ... of one direction.

    With ``n`` buckets to a direction and ``e = n // 2``, distances below ``e``
    have a bucket each; bucket ``e + k`` begins where ``(r / e)^(n - e)``
    reaches ``(max_distance / e)^k``, decided on whole numbers so that no
    rounding of a logarithm moves a border.
    """
    n = num_buckets // 2 if bidirectional else num_buckets
    e = n // 2
    borders = list(range(1, e + 1))
    lo = e
    for k in range(1, n - e):
        want = max_distance ** k * e ** (n - e)
        hi = max_distance
        while lo < hi:  # smallest r with r^(n-e) e^k >= want
            mid = (lo + hi) // 2
            if mid ** (n - e) * e ** k >= want:
                hi = mid
            else:
                lo = mid + 1
        borders.append(lo)
    return tuple(borders)


class BucketBias:
    """A learned bias of relative position: ``table [num_buckets, heads]`` (a CUDA
    tensor, or a numpy array for the forms of ``rvc_cuda.ops``).

    The bias of query ``i`` and key ``j`` is ``table[bucket(j - i), head]``.
    ``bidirectional``: the first half of the rows holds distances of keys at or
    behind the query, the second half those of keys ahead; otherwise every key
    ahead counts as distance 0.  Distances of ``max_distance`` and more share
    the last bucket.  The object holds the table itself (an optimiser may
    change it in place between calls) and the borders of the buckets.
    """

    def __init__(self, table, max_distance: int = 128, bidirectional: bool = True):
        if table.ndim != 2:
            raise ValueError(f"BucketBias: table [num_buckets, heads] expected, got shape {tuple(table.shape)}")
        n, max_distance = int(table.shape[0]), int(max_distance)
        if bidirectional and n % 2:
            raise ValueError(f"BucketBias: {n} buckets cannot be shared by two directions")
        half = n // 2 if bidirectional else n
        if half < 2 or n > MAX_BUCKETS:
            raise ValueError(f"BucketBias: {n} buckets; 2 to {MAX_BUCKETS // (1 + bool(bidirectional))} to a direction "
                             "are supported")
        if not half // 2 < max_distance < 1 << 30:
            raise ValueError(f"BucketBias: max_distance {max_distance} must exceed the {half // 2} single distances")
        self.table = table
        self.num_buckets, self.max_distance, self.bidirectional = n, max_distance, bool(bidirectional)
        b = bucket_borders(n, max_distance, self.bidirectional)
        self._borders = (C.c_int32 * max(1, len(b)))(*b)
        self._nborders = len(b)


def _offset(q_offset) -> int:
    try:
        n = operator.index(q_offset)
    except TypeError:
        raise ValueError(f"q_offset: a whole number is expected, got {q_offset!r}") from None
    if not -(1 << 31) <= n <= 1 << 31:
        raise ValueError(f"q_offset {n} out of range")
    return n


def _length(n) -> int:
    try:
        i = operator.index(n)
    except TypeError:
        i = -1
    if i < 0:
        raise ValueError(f"relative_bias: lengths are whole numbers from 0 on, got {n!r}")
    return i


def _scale(scale, D: int) -> float:
    s = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not abs(s) <= MAX_SCALE:
        raise ValueError(f"attention: scale {s} is not finite in float32")
    return s
