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
_MAX_DIM = _native.CIRCUIT_INT8_MAX_DIM

# A small call is a few microseconds of host time: the current device and its stream are asked for as plain integers
# (torch.cuda.current_stream() builds an object, 3.4 us), and messages are only formatted once a check has failed.
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _cuda(t, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be CUDA tensor")


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """A [n, dim] tensor of values that lie next to each other in each row (a copy if they do not)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be CUDA tensor")
    if t.ndim != 2:
        raise ValueError(f"{name} must have shape [n, dim]")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} asks for a gradient: the 8-bit rows have no backward pass (use torch.no_grad())")
    n, dim = t.shape
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"dim must be in [1, {_MAX_DIM}]")
    s0, s1 = t.stride()
    if (s1 != 1 and dim > 1) or (s0 < dim and n > 1):
        return t.contiguous()
    return t


def _step(t: torch.Tensor) -> int:
    """Elements from one row of a [n, dim] tensor to the next (a single row may carry any number)."""
    n, dim = t.shape
    s = t.stride(0)
    return s if n > 1 or s > dim else dim


def _ids(t: torch.Tensor, name: str, dev: int) -> torch.Tensor:
    _cuda(t, name)
    if t.dtype != torch.int64 and t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32 or int64")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the rows' device")
    return t.contiguous()


def _pair(codes, scales, name: str) -> None:
    """Checks codes [n, dim] int8 and scales [n] float32 of one device."""
    _cuda(codes, name + " codes")
    _cuda(scales, name + " scales")
    if codes.ndim != 2 or codes.dtype != torch.int8:
        raise ValueError(f"{name} codes must be int8 of shape [n, dim]")
    if scales.ndim != 1 or scales.dtype != torch.float32 or scales.shape[0] != codes.shape[0]:
        raise ValueError(f"{name} scales must be float32 of shape [n]")
    if scales.get_device() != codes.get_device():
        raise ValueError(f"{name} codes and scales must be on one device")
    if not 1 <= codes.shape[1] <= _MAX_DIM:
        raise ValueError(f"dim must be in [1, {_MAX_DIM}]")


def _target(t: torch.Tensor, name: str) -> None:
    """Refuses an output whose rows overlap or are not contiguous."""
    n, dim = t.shape
    if (dim > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < dim):
        raise ValueError(f"{name} must be contiguous in each row and its rows must not overlap")


def _quantize(rows, residual, weight, norm, eps, slots, out):
    rows = _rows(rows, "rows")
    dev = rows.get_device()
    if dev != _device():
        with torch.cuda.device(dev):
            return _quantize(rows, residual, weight, norm, eps, slots, out)
    n, dim = rows.shape
    summed = None
    res_ptr = res_step = sum_ptr = w_ptr = slot_ptr = None
    w_type = slot_bytes = 0
    if residual is not None:
        residual = _rows(residual, "residual")
        if residual.shape != rows.shape or residual.dtype != rows.dtype or residual.get_device() != dev:
            raise ValueError("residual must have the shape, type and device of rows")
        summed = torch.empty((n, dim), dtype=rows.dtype, device=rows.device)
        res_ptr, sum_ptr = residual.data_ptr(), summed.data_ptr()
        res_step = _step(residual)
    if weight is not None:
        _cuda(weight, "weight")
        if weight.dtype != rows.dtype and weight.dtype != torch.float32:
            raise ValueError("weight must be of the rows' type or float32")
        if weight.shape != (dim,) or weight.get_device() != dev:
            raise ValueError("weight must have shape [dim] and be on the rows' device")
        if weight.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("weight asks for a gradient: the 8-bit rows have no backward pass (use torch.no_grad())")
        weight = weight.contiguous()
        w_ptr, w_type = weight.data_ptr(), _TYPES[weight.dtype]
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")
    if slots is not None:
        if out is None:
            raise ValueError("slots need the store to write to as out=(codes, scales)")
        slots = _ids(slots, "slots", dev)
        if slots.shape != (n,):
            raise ValueError("slots must have shape [n]")
        slot_ptr, slot_bytes = slots.data_ptr(), slots.element_size()
    if out is None:
        capacity, step = n, (dim + 15) // 16 * 16
        codes = torch.empty((n, step), dtype=torch.int8, device=rows.device)
        scales = torch.empty(n, dtype=torch.float32, device=rows.device)
        if step != dim:
            codes = codes[:, :dim]
    else:
        codes, scales = out
        _pair(codes, scales, "out")
        _target(codes, "out codes")
        if not scales.is_contiguous():
            raise ValueError("out scales must be contiguous")
        if codes.get_device() != dev:
            raise ValueError("out must be on the rows' device")
        capacity, step = codes.shape[0], _step(codes)
        if codes.shape[1] != dim:
            raise ValueError("out must have the rows' dim")
        if slots is None and capacity != n:
            raise ValueError("out must hold as many rows as there are (or give slots)")
    if n and capacity:
        rc = _native.lib().circuit_op_quantize_rows(
            rows.data_ptr(), _TYPES[rows.dtype], n, dim, _step(rows), res_ptr, res_step or 0, w_ptr, w_type, norm, eps,
            sum_ptr, dim, slot_ptr, slot_bytes, capacity, codes.data_ptr(), step, scales.data_ptr(), _stream(dev))
        if rc:
            _native.check(rc, "quantize_rows")
    elif n and summed is not None:  # a store without slots: nothing is written, the sum is still due
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
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    dev = codes.get_device()
    if dev != _device():
        with torch.cuda.device(dev):
            return dequantize_rows(codes, scales, ids, dtype, out)
    rows, dim = codes.shape
    s0, s1 = codes.stride()
    if (s1 != 1 and dim > 1) or (s0 < dim and rows > 1):
        codes = codes.contiguous()
    scales = scales.contiguous()
    n, shape, id_ptr, id_bytes = rows, (rows, dim), None, 0
    if ids is not None:
        ids = _ids(ids, "ids", dev)
        n, shape = ids.numel(), (*ids.shape, dim)
        id_ptr, id_bytes = ids.data_ptr(), ids.element_size()
    step = dim
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=codes.device)
    else:
        _cuda(out, "out")
        if out.dtype != dtype or out.get_device() != dev or out.shape != (n, dim):
            raise ValueError(f"out must be of type dtype, of shape [{n}, {dim}], on the rows' device")
        _target(out, "out")
        step = _step(out)
    if n:
        rc = _native.lib().circuit_op_dequantize_rows(codes.data_ptr(), _step(codes), scales.data_ptr(), rows, dim,
                                                      id_ptr, id_bytes, n, out.data_ptr(), _TYPES[dtype], step,
                                                      _stream(dev))
        if rc:
            _native.check(rc, "dequantize_rows")
    return out


def _code_rows(codes: torch.Tensor) -> torch.Tensor:
    """Codes as the products read them: rows on 16 bytes, their padding inside the storage (a padded copy if not)."""
    n, dim = codes.shape
    step, padded = _step(codes), (dim + 15) // 16 * 16
    if ((dim == 1 or codes.stride(1) == 1) and step % 16 == 0 and step >= padded and codes.data_ptr() % 16 == 0
            and (padded == dim or codes.storage_offset() + (n - 1) * step + padded <= codes.untyped_storage().nbytes())):
        return codes
    return torch.empty((n, padded), dtype=torch.int8, device=codes.device)[:, :dim].copy_(codes)


def int8_scores(query_codes: torch.Tensor, query_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float32,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Products [nq, n] of 8-bit queries with 8-bit rows: query_scales[i] * scales[j] * (codes' inner product), plus
    bias[j] (float32 [n]: a prior of each row, or -|x|^2 / 2 for distances), rounded once to ``dtype``.

    The sum over dim is exact.  Codes whose rows do not start on 16 bytes or end without padding are copied first;
    those of quantize_rows and Int8Rows never are."""
    _pair(query_codes, query_scales, "query")
    _pair(codes, scales, "rows'")
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    dev = codes.get_device()
    if query_codes.get_device() != dev:
        raise ValueError("queries must be on the rows' device")
    if dev != _device():
        with torch.cuda.device(dev):
            return int8_scores(query_codes, query_scales, codes, scales, bias, dtype, out)
    nq, dim = query_codes.shape
    n = codes.shape[0]
    if codes.shape[1] != dim:
        raise ValueError("queries and rows must have one dim")
    if nq > _native.CIRCUIT_INT8_MAX_QUERIES:
        raise ValueError(f"at most {_native.CIRCUIT_INT8_MAX_QUERIES} queries a call")
    bias_ptr = None
    if bias is not None:
        _cuda(bias, "bias")
        if bias.dtype != torch.float32 or bias.shape != (n,) or bias.get_device() != dev:
            raise ValueError("bias must be float32 of shape [n] on the rows' device")
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    step = n
    if out is None:
        out = torch.empty((nq, n), dtype=dtype, device=codes.device)
    else:
        _cuda(out, "out")
        if out.dtype != dtype or out.shape != (nq, n) or out.get_device() != dev:
            raise ValueError(f"out must be of type dtype, of shape [{nq}, {n}], on the rows' device")
        _target(out, "out")
        step = _step(out)
    if nq and n:
        query_codes, codes = _code_rows(query_codes), _code_rows(codes)
        query_scales, scales = query_scales.contiguous(), scales.contiguous()
        rc = _native.lib().circuit_op_int8_scores(
            query_codes.data_ptr(), _step(query_codes), query_scales.data_ptr(), nq, codes.data_ptr(), _step(codes),
            scales.data_ptr(), n, dim, bias_ptr, out.data_ptr(), _TYPES[dtype], step, _stream(dev))
        if rc:
            _native.check(rc, "int8_scores")
    return out
