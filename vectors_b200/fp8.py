"""Rows kept in 8 bits: e4m3 codes with one power-of-two scale for each block of 128 dimensions.

No counterpart in the reference, whose quantizers (SQ8 / SQ4 / BQ / PQ / FP16) encode on the host and
serve only a fused top-k.  These functions work on CUDA tensors that the caller owns:

* ``fp8_empty(capacity, dim)``     a store: codes [capacity][dim rounded up to 128] (float8_e4m3fn)
                                   and scales [capacity][blocks rounded up to 4] (uint8, a byte b
                                   standing for 2^(b - 127), 255 for NaN)
* ``fp8_write_device``             rows quantised into slots of the store as they arrive
* ``fp8_read_device``              stored rows brought back as floats, e.g. a search's candidates
* ``fp8_scores_device``            the full score matrix of a query batch (dot products)
* ``fp8_scores_grouped_device``    each group of queries against its own rows: (query, list) pairs
                                   sorted by list, tokens sorted by expert

A store's rows may be sliced (``codes[a:b], scales[a:b]``), saved or moved like any tensors.  Work is
queued on ``stream`` (a raw handle, default the current stream) and can be captured into a CUDA
graph.  Exceptions are those of the index SPI (``index_spi``).
"""
from __future__ import annotations

import contextlib
from typing import Optional

from . import _native as N
from .index_spi import IllegalArgumentException, NullPointerException, _check

BLOCK = 128


def fp8_pitch(dim: int) -> tuple[int, int]:
    """(bytes of codes, bytes of scales) of one stored row of ``dim`` dimensions."""
    if dim <= 0 or dim > 65536:
        raise IllegalArgumentException(f"dimension must be in [1, 65536]: {dim}")
    blocks = -(-dim // BLOCK)
    return blocks * BLOCK, -(-blocks // 4) * 4


def fp8_empty(capacity: int, dim: int, device="cuda"):
    """A store of ``capacity`` rows of zeros: (codes, scales)."""
    import torch

    if capacity < 0:
        raise IllegalArgumentException(f"capacity must not be negative: {capacity}")
    kp, sp = fp8_pitch(dim)
    codes = torch.zeros((capacity, kp), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    return codes, torch.zeros((capacity, sp), dtype=torch.uint8, device=device)


_TYPES: dict = {}


def _type_of(dtype, name: str) -> int:
    if not _TYPES:
        import torch

        _TYPES.update({torch.float32: N.VX_F32, torch.float16: N.VX_F16, torch.bfloat16: N.VX_BF16})
    t = _TYPES.get(dtype)
    if t is None:
        raise IllegalArgumentException(f"{name} must be float32, float16 or bfloat16, got {dtype}")
    return t


def _store(codes, scales, what: str = "") -> None:
    """codes and scales are one store's contiguous buffers on one GPU."""
    import torch

    if codes is None or scales is None:
        raise NullPointerException(f"{what}codes and {what}scales must not be null")
    if codes.dtype is not torch.float8_e4m3fn and codes.dtype is not torch.uint8:
        raise IllegalArgumentException(f"{what}codes must be float8_e4m3fn or uint8, got {codes.dtype}")
    if scales.dtype is not torch.uint8:
        raise IllegalArgumentException(f"{what}scales must be uint8, got {scales.dtype}")
    if codes.dim() != 2 or scales.dim() != 2 or codes.shape[1] == 0 or codes.shape[1] % BLOCK:
        raise IllegalArgumentException(f"{what}codes must be [rows][a multiple of 128] and {what}scales [rows][...]")
    n, kp = codes.shape
    if tuple(scales.shape) != (n, -(-kp // (4 * BLOCK)) * 4):
        raise IllegalArgumentException(f"{what}scales must be [{n}][{-(-kp // (4 * BLOCK)) * 4}], got {list(scales.shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise IllegalArgumentException(f"{what}codes and {what}scales must be contiguous")
    _on(codes, codes.device, f"{what}codes")
    _on(scales, codes.device, f"{what}scales")


def _on(t, device, name: str) -> None:
    if t.device != device or device.type != "cuda":
        raise IllegalArgumentException(f"{name} must be on the store's CUDA device ({device}), got {t.device}")


def _matrix(t, device, name: str):
    """A 2-D tensor as rows of consecutive elements (a copy where it is laid out otherwise)."""
    if t is None:
        raise NullPointerException(f"{name} must not be null")
    if t.dim() != 2:
        raise IllegalArgumentException(f"{name} must be a 2-D tensor of rows")
    _on(t, device, name)
    n, dim = t.shape
    if (dim > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < dim):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else max(dim, 1))


def _out(out, shape, dtype, device, zero: bool):
    """The result tensor: the caller's, which must have this shape and rows of consecutive elements,
    or a new one of ``dtype`` (float32 if none is given)."""
    import torch

    if out is None:
        return (torch.zeros if zero else torch.empty)(shape, dtype=dtype or torch.float32, device=device)
    if tuple(out.shape) != tuple(shape):
        raise IllegalArgumentException(f"out must be {list(shape)}, got {list(out.shape)}")
    if dtype is not None and out.dtype is not dtype:
        raise IllegalArgumentException(f"out is {out.dtype}, not {dtype}")
    _on(out, device, "out")
    if (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise IllegalArgumentException("out must have rows of consecutive elements that do not overlap")
    return out


def _slots(slots, device):
    """(pointer, bytes per slot, tensor kept alive) of a slot list."""
    import torch

    if slots.dtype is not torch.int64 and slots.dtype is not torch.int32:
        raise IllegalArgumentException(f"slots must be int32 or int64, got {slots.dtype}")
    if slots.dim() != 1:
        raise IllegalArgumentException("slots must be a 1-D tensor")
    _on(slots, device, "slots")
    slots = slots.contiguous()
    return slots.data_ptr(), slots.element_size(), slots


def _queue(device, stream):
    """The raw stream handle, and a context in which tensors are allocated and copied on it."""
    import torch

    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream, contextlib.nullcontext()
    return stream, torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def fp8_write_device(rows, codes, scales, slots=None, first: int = 0, stream=None) -> None:
    """Quantises rows [n][dim] (float32 / float16 / bfloat16) into a store: row i into slot
    ``slots[i]`` (int32 or int64; outside [0, capacity) the row is skipped; of rows that name the same
    slot the last is kept), or into ``first + i`` without slots.  Other rows stay as they are.  Writes
    that overlap on other streams are ordered by the caller."""
    _store(codes, scales)
    device = codes.device
    st, queue = _queue(device, stream)
    with queue:
        rows, stride = _matrix(rows, device, "rows")
        n, dim = rows.shape
        if fp8_pitch(dim)[0] != codes.shape[1]:
            raise IllegalArgumentException(f"rows of dimension {dim} do not match the store's {codes.shape[1]} columns")
        ptr, size, kept = (None, 8, None) if slots is None else _slots(slots, device)
        if slots is not None and len(slots) != n:
            raise IllegalArgumentException(f"slots must be [{n}], got {list(slots.shape)}")
        _check(N.lib().vx_fp8_write_device(device.index, rows.data_ptr(), _type_of(rows.dtype, "rows"), n, dim, stride, ptr,
                                           size, first, codes.data_ptr(), scales.data_ptr(), codes.shape[0], st))


def fp8_read_device(codes, scales, dim: int, slots=None, first: int = 0, count: Optional[int] = None, dtype=None,
                    out=None, stream=None):
    """Stored rows as floats [n][dim] (``dtype`` float32, float16 or bfloat16): those of ``slots``
    (int32 or int64, of any search result; outside [0, capacity) a row of zeros), or ``count`` rows
    from ``first`` (default: to the end)."""
    _store(codes, scales)
    if fp8_pitch(dim)[0] != codes.shape[1]:
        raise IllegalArgumentException(f"dimension {dim} does not match the store's {codes.shape[1]} columns")
    device = codes.device
    st, queue = _queue(device, stream)
    with queue:
        ptr, size, kept = (None, 8, None) if slots is None else _slots(slots, device)
        n = len(slots) if slots is not None else codes.shape[0] - first if count is None else count
        if n < 0 or (slots is not None and count not in (None, n)):
            raise IllegalArgumentException(f"count {count} does not match the {n} rows asked for")
        out = _out(out, (n, dim), dtype, device, False)
        stride = out.stride(0) if n > 1 else dim
        _check(N.lib().vx_fp8_read_device(device.index, codes.data_ptr(), scales.data_ptr(), codes.shape[0], dim, ptr, size,
                                          first, n, out.data_ptr(), _type_of(out.dtype, "out"), stride, st))
    return out


def _queries(queries, query_scales, codes):
    """(tensor, type, pointer of its scales, stride, dim) of float or stored queries."""
    if queries is None:
        raise NullPointerException("queries must not be null")
    if query_scales is not None:
        _store(queries, query_scales, "query ")
        _on(queries, codes.device, "queries")
        if queries.shape[1] != codes.shape[1]:
            raise IllegalArgumentException(f"queries of {queries.shape[1]} columns do not match the store's {codes.shape[1]}")
        return queries, N.VX_E4M3, query_scales.data_ptr(), queries.shape[1], queries.shape[1]
    queries, stride = _matrix(queries, codes.device, "queries")
    dim = queries.shape[1]
    if fp8_pitch(dim)[0] != codes.shape[1]:
        raise IllegalArgumentException(f"Query dimension {dim} does not match the store's {codes.shape[1]} columns")
    return queries, _type_of(queries.dtype, "queries"), None, stride, dim


def fp8_scores_device(queries, codes, scales, query_scales=None, dtype=None, out=None, stream=None):
    """dot(query, row) of every query and stored row: [nq][rows] of ``dtype`` (float32, float16 or
    bfloat16), into ``out`` if given.  Queries are floats [nq][dim], quantised as stored rows are, or
    stored rows themselves (codes, with their ``query_scales``)."""
    _store(codes, scales)
    device = codes.device
    st, queue = _queue(device, stream)
    with queue:
        q, qtype, qs, stride, dim = _queries(queries, query_scales, codes)
        nq, n = q.shape[0], codes.shape[0]
        if nq == 0:
            raise IllegalArgumentException("queries must not be empty")
        out = _out(out, (nq, n), dtype, device, False)
        ldo = out.stride(0) if nq > 1 else max(n, 1)
        _check(N.lib().vx_fp8_scores_device(device.index, q.data_ptr(), qtype, qs, nq, stride, codes.data_ptr(),
                                            scales.data_ptr(), n, dim, out.data_ptr(), _type_of(out.dtype, "out"), ldo, st))
    return out


def fp8_scores_grouped_device(queries, query_offsets, codes, scales, row_offsets, query_scales=None,
                              max_rows: Optional[int] = None, dtype=None, out=None, stream=None):
    """For each group g the products of queries ``query_offsets[g]:query_offsets[g + 1]`` with stored rows
    ``row_offsets[g]:row_offsets[g + 1]`` (int64 CUDA tensors [groups + 1]; sizes may differ or be zero):
    out[i][j] for the group's j-th row, [nq][max_rows].  Without ``out`` the result is new and zero
    past each group's rows; in a given ``out`` (whose width is max_rows) those values, and rows of
    queries in no group, stay as they are.  A group's rows past max_rows are not scored."""
    import torch

    _store(codes, scales)
    device = codes.device
    st, queue = _queue(device, stream)
    with queue:
        q, qtype, qs, stride, dim = _queries(queries, query_scales, codes)
        for t, name in ((query_offsets, "query_offsets"), (row_offsets, "row_offsets")):
            if t is None:
                raise NullPointerException(f"{name} must not be null")
            if t.dtype is not torch.int64 or t.dim() != 1 or len(t) == 0 or not t.is_contiguous():
                raise IllegalArgumentException(f"{name} must be a contiguous int64 tensor of groups + 1 offsets")
            _on(t, device, name)
        if len(query_offsets) != len(row_offsets):
            raise IllegalArgumentException(
                f"query_offsets and row_offsets differ in length: {len(query_offsets)} and {len(row_offsets)}")
        if out is not None and out.dim() == 2 and max_rows is None:
            max_rows = out.shape[1]
        if max_rows is None or max_rows < 0:
            raise IllegalArgumentException("max_rows or out must be given")
        nq = q.shape[0]
        out = _out(out, (nq, max_rows), dtype, device, True)
        ldo = out.stride(0) if nq > 1 else max(max_rows, 1)
        _check(N.lib().vx_fp8_scores_grouped_device(device.index, q.data_ptr(), qtype, qs, nq, stride,
                                                    query_offsets.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                                                    codes.shape[0], row_offsets.data_ptr(), len(row_offsets) - 1, dim,
                                                    out.data_ptr(), _type_of(out.dtype, "out"), ldo, max_rows, st))
    return out


def fp8_check(device: int = 0, stream=None) -> None:
    """Waits for the stream and raises if a bounded wait inside a score product has run out."""
    import torch

    st = torch.cuda.current_stream(device).cuda_stream if stream is None else stream
    _check(N.lib().vx_fp8_check(device, st))
