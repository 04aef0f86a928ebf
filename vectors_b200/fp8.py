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

import functools
from typing import Optional

import torch

from . import _native as N
from .index_spi import IllegalArgumentException, NullPointerException, _check

BLOCK = 128

_TYPES = {torch.float32: N.VX_F32, torch.float16: N.VX_F16, torch.bfloat16: N.VX_BF16}
_CODES = (torch.float8_e4m3fn, torch.uint8)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # none without CUDA: no store gets that far


@functools.lru_cache(maxsize=None)
def _call(name: str):
    return getattr(N.lib(), name)


def fp8_pitch(dim: int) -> tuple[int, int]:
    """(bytes of codes, bytes of scales) of one stored row of ``dim`` dimensions."""
    if dim <= 0 or dim > 65536:
        raise IllegalArgumentException(f"dimension must be in [1, 65536]: {dim}")
    blocks = -(-dim // BLOCK)
    return blocks * BLOCK, -(-blocks // 4) * 4


def fp8_empty(capacity: int, dim: int, device="cuda"):
    """A store of ``capacity`` rows of zeros: (codes, scales)."""
    if capacity < 0:
        raise IllegalArgumentException(f"capacity must not be negative: {capacity}")
    kp, sp = fp8_pitch(dim)
    codes = torch.zeros((capacity, kp), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    return codes, torch.zeros((capacity, sp), dtype=torch.uint8, device=device)


def _type_of(t, name: str) -> int:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise IllegalArgumentException(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return kind


def _store(codes, scales, what: str = ""):
    """(rows, columns, device number) of a store: contiguous buffers on one GPU."""
    if codes is None or scales is None:
        raise NullPointerException(f"{what}codes and {what}scales must not be null")
    if codes.dtype not in _CODES:
        raise IllegalArgumentException(f"{what}codes must be float8_e4m3fn or uint8, got {codes.dtype}")
    if scales.dtype is not torch.uint8:
        raise IllegalArgumentException(f"{what}scales must be uint8, got {scales.dtype}")
    shape = codes.shape
    if len(shape) != 2 or shape[1] == 0 or shape[1] % BLOCK:
        raise IllegalArgumentException(f"{what}codes must be [rows][a multiple of 128], got {list(shape)}")
    n, kp = shape
    if scales.shape != (n, -(-kp // (4 * BLOCK)) * 4):
        raise IllegalArgumentException(f"{what}scales must be [{n}][{-(-kp // (4 * BLOCK)) * 4}], got {list(scales.shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise IllegalArgumentException(f"{what}codes and {what}scales must be contiguous")
    device = codes.get_device()
    if device < 0:
        raise IllegalArgumentException(f"{what}codes must be on a CUDA device, got {codes.device}")
    _on(scales, device, "scales")
    return n, kp, device


def _on(t, device: int, name: str) -> None:
    if t.get_device() != device:
        raise IllegalArgumentException(f"{name} must be on the store's CUDA device ({device}), got {t.device}")


def _matrix(t, device: int, name: str):
    """A 2-D tensor as rows of consecutive elements (a copy where it is laid out otherwise), its shape
    and the elements from one row to the next."""
    if t is None:
        raise NullPointerException(f"{name} must not be null")
    if t.dim() != 2:
        raise IllegalArgumentException(f"{name} must be a 2-D tensor of rows")
    _on(t, device, name)
    n, dim = t.shape
    step, by = t.stride()
    # negated views (the imaginary part of a conjugate) have steps of two: only single columns need asking
    if (dim > 1 and by != 1) or (n > 1 and step < dim) or (dim == 1 and t.is_neg()):
        t, step = t.resolve_neg().contiguous(), dim
    return t, n, dim, step if n > 1 else dim


def _out(out, rows: int, columns: int, dtype, codes, zero: bool):
    """The result tensor (the caller's, which must have this shape and rows of consecutive elements that do
    not overlap, or a new one of ``dtype``, float32 if none is given) and the elements between its rows."""
    if out is None:
        if zero:
            return codes.new_zeros((rows, columns), dtype=dtype or torch.float32), columns
        # the quickest of torch's ways to a new tensor (1.5 us; new_empty 2.0)
        return torch.empty_strided((rows, columns), (columns, 1), dtype=dtype or torch.float32, device=codes.device), columns
    if out.shape != (rows, columns):
        raise IllegalArgumentException(f"out must be {[rows, columns]}, got {list(out.shape)}")
    if dtype is not None and out.dtype is not dtype:
        raise IllegalArgumentException(f"out is {out.dtype}, not {dtype}")
    _on(out, codes.get_device(), "out")
    step, by = out.stride()
    if (columns > 1 and by != 1) or (rows > 1 and step < columns):
        raise IllegalArgumentException("out must have rows of consecutive elements that do not overlap")
    if columns == 1 and out.is_neg():
        raise IllegalArgumentException("out must not be a negated view")
    return out, step if rows > 1 else columns


def _slots(slots, device: int):
    """A slot list as consecutive int32 or int64."""
    if slots.dtype is not torch.int64 and slots.dtype is not torch.int32:
        raise IllegalArgumentException(f"slots must be int32 or int64, got {slots.dtype}")
    if slots.dim() != 1:
        raise IllegalArgumentException("slots must be a 1-D tensor")
    _on(slots, device, "slots")
    return slots.contiguous()


def _place(first: int, n: int, capacity: int, slots) -> None:
    """Rows first .. first + n - 1 must lie in the store (the library's check sees 64 bits of a number); with
    slots there is no first row."""
    if slots is not None:
        raise IllegalArgumentException(f"first ({first}) and slots exclude each other")
    if first < 0 or n > capacity - first:
        raise IllegalArgumentException(f"rows [{first}, {first + n}) do not fit a store of {capacity}")


def _on_stream(stream: int, codes):
    """Makes a raw stream current, so that what a call allocates or copies belongs to it."""
    device = codes.get_device() if isinstance(codes, torch.Tensor) and codes.is_cuda else None
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def fp8_write_device(rows, codes, scales, slots=None, first: int = 0, stream=None) -> None:
    """Quantises rows [n][dim] (float32 / float16 / bfloat16) into a store: row i into slot
    ``slots[i]`` (int32 or int64; outside [0, capacity) the row is skipped; of rows that name the same
    slot the last is kept), or into ``first + i`` (``first`` is for calls without slots).  Other rows stay as they are.  Writes
    that overlap on other streams are ordered by the caller."""
    if stream is not None:
        with _on_stream(stream, codes):
            return fp8_write_device(rows, codes, scales, slots, first)
    capacity, kp, device = _store(codes, scales)
    rows, n, dim, step = _matrix(rows, device, "rows")
    if dim > kp or dim <= kp - BLOCK:
        raise IllegalArgumentException(f"rows of dimension {dim} do not match the store's {kp} columns")
    at, size = None, 8
    if slots is not None:
        slots = _slots(slots, device)
        if slots.shape[0] != n:
            raise IllegalArgumentException(f"slots must be [{n}], got {list(slots.shape)}")
        at, size = slots.data_ptr(), slots.element_size()
    if first != 0:
        _place(first, n, capacity, slots)
    _check(_call("vx_fp8_write_device")(device, rows.data_ptr(), _type_of(rows, "rows"), n, dim, step, at, size, first,
                                        codes.data_ptr(), scales.data_ptr(), capacity, _raw_stream(device)))


def fp8_read_device(codes, scales, dim: int, slots=None, first: int = 0, count: Optional[int] = None, dtype=None,
                    out=None, stream=None):
    """Stored rows as floats [n][dim] (``dtype`` float32, float16 or bfloat16): those of ``slots``
    (int32 or int64, of any search result; outside [0, capacity) a row of zeros), or ``count`` rows
    from ``first`` (default: to the end)."""
    if stream is not None:
        with _on_stream(stream, codes):
            return fp8_read_device(codes, scales, dim, slots, first, count, dtype, out)
    capacity, kp, device = _store(codes, scales)
    if dim > kp or dim <= kp - BLOCK:
        raise IllegalArgumentException(f"dimension {dim} does not match the store's {kp} columns")
    at, size = None, 8
    if slots is not None:
        slots = _slots(slots, device)
        at, size, n = slots.data_ptr(), slots.element_size(), slots.shape[0]
    else:
        n = capacity - first if count is None else count
    if n < 0 or (count is not None and count != n):
        raise IllegalArgumentException(f"count {count} does not match the {n} rows asked for")
    if first != 0:
        _place(first, n, capacity, slots)
    out, step = _out(out, n, dim, dtype, codes, False)
    _check(_call("vx_fp8_read_device")(device, codes.data_ptr(), scales.data_ptr(), capacity, dim, at, size, first, n,
                                       out.data_ptr(), _type_of(out, "out"), step, _raw_stream(device)))
    return out


def _queries(queries, query_scales, kp: int, device: int):
    """(tensor, count, dim, type, pointer of its scales, elements between rows) of float or stored queries."""
    if query_scales is not None:
        nq, columns, on = _store(queries, query_scales, "query ")
        if on != device or columns != kp:
            raise IllegalArgumentException(f"queries of {columns} columns on device {on} do not match the store's {kp} on {device}")
        return queries, nq, kp, N.VX_E4M3, query_scales.data_ptr(), kp
    queries, nq, dim, step = _matrix(queries, device, "queries")
    if dim > kp or dim <= kp - BLOCK:
        raise IllegalArgumentException(f"Query dimension {dim} does not match the store's {kp} columns")
    return queries, nq, dim, _type_of(queries, "queries"), None, step


def fp8_scores_device(queries, codes, scales, query_scales=None, dtype=None, out=None, stream=None):
    """dot(query, row) of every query and stored row: [nq][rows] of ``dtype`` (float32, float16 or
    bfloat16), into ``out`` if given.  Queries are floats [nq][dim], quantised as stored rows are, or
    stored rows themselves (codes, with their ``query_scales``)."""
    if stream is not None:
        with _on_stream(stream, codes):
            return fp8_scores_device(queries, codes, scales, query_scales, dtype, out)
    n, kp, device = _store(codes, scales)
    q, nq, dim, kind, qs, step = _queries(queries, query_scales, kp, device)
    if nq == 0:
        raise IllegalArgumentException("queries must not be empty")
    out, ldo = _out(out, nq, n, dtype, codes, False)
    _check(_call("vx_fp8_scores_device")(device, q.data_ptr(), kind, qs, nq, step, codes.data_ptr(), scales.data_ptr(), n,
                                         dim, out.data_ptr(), _type_of(out, "out"), ldo, _raw_stream(device)))
    return out


def _offsets(t, device: int, name: str) -> int:
    if t is None:
        raise NullPointerException(f"{name} must not be null")
    if t.dtype is not torch.int64 or t.dim() != 1 or t.shape[0] == 0 or not t.is_contiguous():
        raise IllegalArgumentException(f"{name} must be a contiguous int64 tensor of groups + 1 offsets")
    _on(t, device, name)
    return t.shape[0] - 1


def fp8_scores_grouped_device(queries, query_offsets, codes, scales, row_offsets, query_scales=None,
                              max_rows: Optional[int] = None, dtype=None, out=None, stream=None):
    """For each group g the products of queries ``query_offsets[g]:query_offsets[g + 1]`` with stored rows
    ``row_offsets[g]:row_offsets[g + 1]`` (int64 CUDA tensors [groups + 1]; sizes may differ or be zero):
    out[i][j] for the group's j-th row, [nq][max_rows].  Without ``out`` the result is new and zero
    past each group's rows; in a given ``out`` (whose width is max_rows) those values, and rows of
    queries in no group, stay as they are.  A group's rows past max_rows are not scored."""
    if stream is not None:
        with _on_stream(stream, codes):
            return fp8_scores_grouped_device(queries, query_offsets, codes, scales, row_offsets, query_scales, max_rows,
                                             dtype, out)
    n, kp, device = _store(codes, scales)
    q, nq, dim, kind, qs, step = _queries(queries, query_scales, kp, device)
    groups = _offsets(query_offsets, device, "query_offsets")
    if _offsets(row_offsets, device, "row_offsets") != groups:
        raise IllegalArgumentException(
            f"query_offsets and row_offsets differ in length: {groups + 1} and {row_offsets.shape[0]}")
    if out is not None and max_rows is None and out.dim() == 2:
        max_rows = out.shape[1]
    if max_rows is None or max_rows < 0:
        raise IllegalArgumentException("max_rows or out must be given")
    out, ldo = _out(out, nq, max_rows, dtype, codes, True)
    _check(_call("vx_fp8_scores_grouped_device")(device, q.data_ptr(), kind, qs, nq, step, query_offsets.data_ptr(),
                                                 codes.data_ptr(), scales.data_ptr(), n, row_offsets.data_ptr(), groups,
                                                 dim, out.data_ptr(), _type_of(out, "out"), ldo, max_rows,
                                                 _raw_stream(device)))
    return out


def fp8_check(device: int = 0, stream=None) -> None:
    """Waits for the stream and raises if a bounded wait inside a score product has run out."""
    if stream is None:  # a device that is not there has no current stream, and the library says so
        stream = _raw_stream(device) if 0 <= device < torch.cuda.device_count() else 0
    _check(_call("vx_fp8_check")(device, stream))
