"""Rows in 8 bits: quantisation (plain, to unit length, or after a root-mean-square norm with the residual's addition),
a store of such rows, and the products of queries with them.

A row of ``dim`` values is kept as ``dim`` int8 codes and one float32 scale: a quarter of the bytes of the float32 rows
that a CircuitIndex scans.  The products are exact sums of the codes, so they equal the inner products of the rows as
stored; against the original rows each value is off by at most half a code (scale / 2).

The calls run on the current torch stream of their tensors' device, never synchronise, and may be captured into a CUDA
graph.  They serve only: there is no backward pass, and rows that ask for a gradient are refused.  No reference
counterpart (the reference keeps float32 rows only).
"""
from typing import Optional, Tuple

import torch

from circuit_rag import _native

_TYPES = {torch.float32: _native.CIRCUIT_F32, torch.float16: _native.CIRCUIT_F16,
          torch.bfloat16: _native.CIRCUIT_BF16}


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _cuda(t, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be CUDA tensor")


def _rows(t: torch.Tensor, name: str, dtype=None) -> torch.Tensor:
    """A [n, dim] tensor whose values lie next to each other in each row (a copy if they do not)."""
    _cuda(t, name)
    _need(t.ndim == 2, f"{name} must have shape [n, dim]")
    if dtype is None:
        _need(t.dtype in _TYPES, f"{name} must be float32, float16 or bfloat16")
    else:
        _need(t.dtype == dtype, f"{name} must be {str(dtype).replace('torch.', '')}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} asks for a gradient: the 8-bit rows have no backward pass (use torch.no_grad())")
    n, dim = t.shape
    _need(1 <= dim <= _native.CIRCUIT_INT8_MAX_DIM, f"dim must be in [1, {_native.CIRCUIT_INT8_MAX_DIM}]")
    if (dim > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < dim):
        return t.contiguous()
    return t


def _stride(t: torch.Tensor) -> int:
    """Elements from one row to the next (a single row may carry any number)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _padded(dim: int) -> int:
    return (dim + 15) // 16 * 16


def _alloc(n: int, dim: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    codes = torch.empty((n, _padded(dim)), dtype=torch.int8, device=device)
    return (codes if codes.shape[1] == dim else codes[:, :dim]), torch.empty(n, dtype=torch.float32, device=device)


def _ids(t: torch.Tensor, name: str, device) -> torch.Tensor:
    _cuda(t, name)
    _need(t.dtype in (torch.int32, torch.int64), f"{name} must be int32 or int64")
    _need(t.device == device, f"{name} must be on {device}")
    return t.contiguous()


def _pair(codes, scales, name: str, writable: bool = False) -> None:
    """Checks codes [n, dim] int8 and scales [n] float32 of one device."""
    _cuda(codes, name + " codes")
    _cuda(scales, name + " scales")
    _need(codes.ndim == 2 and codes.dtype == torch.int8, f"{name} codes must be int8 of shape [n, dim]")
    _need(scales.ndim == 1 and scales.dtype == torch.float32 and scales.shape[0] == codes.shape[0],
          f"{name} scales must be float32 of shape [n]")
    _need(scales.device == codes.device, f"{name} codes and scales must be on one device")
    if writable:
        _need(codes.shape[1] == 1 or codes.stride(1) == 1, f"{name} codes must be contiguous in each row")
        _need(codes.shape[0] < 2 or codes.stride(0) >= codes.shape[1], f"{name} code rows must not overlap")
        _need(scales.is_contiguous(), f"{name} scales must be contiguous")


class _on:
    """The tensor's device as the current one, and its current stream."""

    __slots__ = ("device", "guard", "stream")

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.guard = None
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _quantize(rows, residual, weight, norm, eps, slots, out):
    rows = _rows(rows, "rows")
    n, dim = rows.shape
    dev = rows.device
    summed = None
    if residual is not None:
        residual = _rows(residual, "residual", rows.dtype)
        _need(residual.shape == rows.shape, "residual must have the shape of rows")
        _need(residual.device == dev, f"residual must be on {dev}")
    if weight is not None:
        _cuda(weight, "weight")
        _need(weight.dtype in (rows.dtype, torch.float32), "weight must be of the rows' type or float32")
        _need(weight.shape == (dim,) and weight.device == dev, f"weight must have shape [dim] and be on {dev}")
        if weight.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("weight asks for a gradient: the 8-bit rows have no backward pass (use torch.no_grad())")
        weight = weight.contiguous()
    _need(0.0 <= eps < float("inf"), "eps must be finite and not negative")
    if slots is not None:
        _need(out is not None, "slots need the store to write to as out=(codes, scales)")
        slots = _ids(slots, "slots", dev)
        _need(slots.shape == (n,), "slots must have shape [n]")
    with _on(dev) as stream:
        if out is None:
            codes, scales = _alloc(n, dim, dev)
        else:
            codes, scales = out
            _pair(codes, scales, "out", writable=True)
            _need(codes.device == dev, f"out must be on {dev}")
            _need(codes.shape[1] == dim, "out must have the rows' dim")
            _need(slots is not None or codes.shape[0] == n, "out must hold as many rows as there are (or give slots)")
        if residual is not None:
            summed = torch.empty((n, dim), dtype=rows.dtype, device=dev)
        if n and codes.shape[0]:
            rc = _native.lib().circuit_op_quantize_rows(
                rows.data_ptr(), _TYPES[rows.dtype], n, dim, _stride(rows),
                residual.data_ptr() if residual is not None else None,
                _stride(residual) if residual is not None else 0,
                weight.data_ptr() if weight is not None else None, _TYPES[weight.dtype] if weight is not None else 0,
                norm, eps, summed.data_ptr() if summed is not None else None, dim,
                slots.data_ptr() if slots is not None else None, slots.element_size() if slots is not None else 0,
                codes.shape[0], codes.data_ptr(), _stride(codes), scales.data_ptr(), stream)
            _native.check(rc, "quantize_rows")
        elif summed is not None and n:
            torch.add(rows, residual, out=summed)
    return codes, scales, summed


def quantize_rows(rows: torch.Tensor, slots: Optional[torch.Tensor] = None,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                  normalize: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """8-bit codes [n, dim] and scales [n] of rows [n, dim] (float32, float16, bfloat16).

    code = rint(127 x / max|x|) of the real quotient, ties to even; scale = max|x| / 127, with ``normalize`` over the
    row's length, so that the stored rows have unit length (products are cosines).  A row of zeros gets scale 0; one
    with an infinity or NaN gets codes 0 and scale NaN, so every product with it is NaN.

    ``out=(codes, scales)`` is written instead of new tensors.  With ``slots`` [n] (int32 or int64) row i goes to row
    slots[i] of ``out``: slots outside it write nothing, of equal slots the last row stays, other rows are left alone.
    New codes are a view of rows padded to a multiple of 16 bytes, as int8_scores reads them."""
    norm = _native.CIRCUIT_NORM_UNIT if normalize else _native.CIRCUIT_NORM_NONE
    return _quantize(rows, None, None, norm, 0.0, slots, out)[:2]


def rms_norm_quantize(rows: torch.Tensor, residual: Optional[torch.Tensor] = None,
                      weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                      slots: Optional[torch.Tensor] = None,
                      out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """Root-mean-square norm of rows + residual, as 8-bit rows: (codes, scales, summed).

    v = rows + residual, rounded once to the rows' type and returned as ``summed`` (None without a residual); the codes
    and scales are those of v / sqrt(mean(v^2) + eps) * weight (weight of the rows' type or float32, or none).  The
    sum of squares is held in 32 bits and cancels in the codes.  ``slots`` and ``out`` as in quantize_rows."""
    return _quantize(rows, residual, weight, _native.CIRCUIT_NORM_RMS, float(eps), slots, out)


def dequantize_rows(codes: torch.Tensor, scales: torch.Tensor, ids: Optional[torch.Tensor] = None,
                    dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values codes * scales [n, dim] of rows ``ids`` (int32 or int64, any shape: the result has shape
    [*ids.shape, dim]; all rows without ids), rounded once to ``dtype``.  A negative id, as a search returns for a
    place without a result, gives zeros; an id past the last row gives NaN."""
    _pair(codes, scales, "rows'")
    _need(dtype in _TYPES, "dtype must be float32, float16 or bfloat16")
    rows, dim = codes.shape
    dev = codes.device
    _need(1 <= dim <= _native.CIRCUIT_INT8_MAX_DIM, f"dim must be in [1, {_native.CIRCUIT_INT8_MAX_DIM}]")
    if (dim > 1 and codes.stride(1) != 1) or (rows > 1 and codes.stride(0) < dim):
        codes = codes.contiguous()
    scales = scales.contiguous()
    if ids is not None:
        ids = _ids(ids, "ids", dev)
    shape = (rows if ids is None else ids.numel(), dim)
    with _on(dev) as stream:
        if out is None:
            out = torch.empty(shape if ids is None else (*ids.shape, dim), dtype=dtype, device=dev)
            flat = out
        else:
            _cuda(out, "out")
            _need(out.dtype == dtype and out.device == dev and out.shape == shape,
                  f"out must be of type dtype, of shape [{shape[0]}, {dim}], on {dev}")
            _need((dim == 1 or out.stride(1) == 1) and (shape[0] < 2 or out.stride(0) >= dim),
                  "out must be contiguous in each row and its rows must not overlap")
            flat = out
        if shape[0]:
            rc = _native.lib().circuit_op_dequantize_rows(
                codes.data_ptr(), _stride(codes), scales.data_ptr(), rows, dim,
                ids.data_ptr() if ids is not None else None, ids.element_size() if ids is not None else 0, shape[0],
                flat.data_ptr(), _TYPES[dtype], _stride(flat) if flat.ndim == 2 else dim, stream)
            _native.check(rc, "dequantize_rows")
    return out


def _code_rows(codes: torch.Tensor) -> torch.Tensor:
    """Codes as int8_scores reads them: rows on 16 bytes, their padding inside the storage (a padded copy if not)."""
    n, dim = codes.shape
    stride = _stride(codes)
    if ((dim == 1 or codes.stride(1) == 1) and stride % 16 == 0 and stride >= _padded(dim)
            and codes.data_ptr() % 16 == 0
            and codes.storage_offset() + (n - 1) * stride + _padded(dim) <= codes.untyped_storage().nbytes()):
        return codes
    new = torch.empty((n, _padded(dim)), dtype=torch.int8, device=codes.device)[:, :dim]
    return new.copy_(codes)


def int8_scores(query_codes: torch.Tensor, query_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float32,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Products [nq, n] of 8-bit queries with 8-bit rows: query_scales[i] * scales[j] * (codes' inner product), plus
    bias[j] (float32 [n]: a prior of each row, or -|x|^2 / 2 for distances), rounded once to ``dtype``.

    The sum over dim is exact.  Codes whose rows do not start on 16 bytes or end without padding are copied first;
    those of quantize_rows and Int8Rows never are."""
    _pair(query_codes, query_scales, "query")
    _pair(codes, scales, "rows'")
    _need(dtype in _TYPES, "dtype must be float32, float16 or bfloat16")
    nq, dim = query_codes.shape
    n = codes.shape[0]
    dev = codes.device
    _need(codes.shape[1] == dim, "queries and rows must have one dim")
    _need(1 <= dim <= _native.CIRCUIT_INT8_MAX_DIM, f"dim must be in [1, {_native.CIRCUIT_INT8_MAX_DIM}]")
    _need(nq <= _native.CIRCUIT_INT8_MAX_QUERIES, f"at most {_native.CIRCUIT_INT8_MAX_QUERIES} queries a call")
    _need(query_codes.device == dev, f"queries must be on {dev}")
    if bias is not None:
        _cuda(bias, "bias")
        _need(bias.dtype == torch.float32 and bias.shape == (n,) and bias.device == dev,
              f"bias must be float32 of shape [n] on {dev}")
        bias = bias.contiguous()
    with _on(dev) as stream:
        if out is None:
            out = torch.empty((nq, n), dtype=dtype, device=dev)
        else:
            _cuda(out, "out")
            _need(out.dtype == dtype and out.shape == (nq, n) and out.device == dev,
                  f"out must be of type dtype, of shape [{nq}, {n}], on {dev}")
            _need((n < 2 or out.stride(1) == 1) and (nq < 2 or out.stride(0) >= n),
                  "out must be contiguous in each row and its rows must not overlap")
        if nq and n:
            query_codes, codes = _code_rows(query_codes), _code_rows(codes)
            query_scales, scales = query_scales.contiguous(), scales.contiguous()
            rc = _native.lib().circuit_op_int8_scores(
                query_codes.data_ptr(), _stride(query_codes), query_scales.data_ptr(), nq, codes.data_ptr(),
                _stride(codes), scales.data_ptr(), n, dim, bias.data_ptr() if bias is not None else None,
                out.data_ptr(), _TYPES[dtype], _stride(out), stream)
            _native.check(rc, "int8_scores")
    return out
