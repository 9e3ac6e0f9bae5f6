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

_bound = None


def _bind():
    """The binding (circuit_rag._int8: checks, outputs and launches of these calls), loaded on first use."""
    global _bound
    if _bound is None:
        _native.lib()  # a missing library is reported as for every other call
        try:
            from circuit_rag import _int8
        except ImportError as e:
            raise _native.NativeLibraryError(f"circuit_rag._int8 cannot be loaded ({e}): build it with "
                                             "`make -C circuit-rag_b200/csrc`") from e
        _bound = _int8
    return _bound


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
    return _bind().quantize(rows, None, None, norm, 0.0, slots, out)


def rms_norm_quantize(rows: torch.Tensor, residual: Optional[torch.Tensor] = None,
                      weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                      slots: Optional[torch.Tensor] = None,
                      out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """Root-mean-square norm of rows + residual, as 8-bit rows: (codes, scales, summed).

    v = rows + residual, rounded once to the rows' type and returned as ``summed`` (None without a residual); the codes
    and scales are those of v / sqrt(mean(v^2) + eps) * weight (weight of the rows' type or float32, or none).  The
    sum of squares is held in 32 bits and cancels in the codes.  ``slots`` and ``out`` as in quantize_rows."""
    return _bind().quantize(rows, residual, weight, _native.CIRCUIT_NORM_RMS, eps, slots, out)


def dequantize_rows(codes: torch.Tensor, scales: torch.Tensor, ids: Optional[torch.Tensor] = None,
                    dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values codes * scales [n, dim] of rows ``ids`` (int32 or int64, any shape: the result has shape
    [*ids.shape, dim]; all rows without ids), rounded once to ``dtype``.  A negative id, as a search returns for a
    place without a result, gives zeros; an id past the last row gives NaN."""
    return _bind().dequantize(codes, scales, ids, dtype, out)


def int8_scores(query_codes: torch.Tensor, query_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float32,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Products [nq, n] of 8-bit queries with 8-bit rows: query_scales[i] * scales[j] * (codes' inner product), plus
    bias[j] (float32 [n]: a prior of each row, or -|x|^2 / 2 for distances), rounded once to ``dtype``.

    The sum over dim is exact.  The rows of a new result start on 128 bytes (its row stride is n rounded up, so it is
    only contiguous where n allows); ``out`` may have any row stride.  Codes whose rows do not start on 16 bytes or end without padding are copied first;
    those of quantize_rows and Int8Rows never are."""
    return _bind().scores(query_codes, query_scales, codes, scales, bias, dtype, out)
