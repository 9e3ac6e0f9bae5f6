"""Rows in 8 bits: quantisation (plain, to unit length, or after a root-mean-square norm with the residual's addition),
a store of such rows, and the products of queries with them.

A row of ``dim`` values is kept as ``dim`` int8 codes and one float32 scale: a quarter of the bytes of the float32 rows
that a CircuitIndex scans.  The products sum the codes exactly, so up to the roundings of the scales they are the inner
products of the rows as stored; against the original rows each value is off by at most half a code (scale / 2).

The calls run on the current torch stream of their tensors' device, never synchronise, and may be captured into a CUDA
graph.  They serve only: there is no backward pass, and tensors that ask for a gradient or carry a forward one are
refused.  Given results count as written in place.  No reference counterpart (the reference keeps float32 rows only).
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
    sum of squares is held in 32 bits and cancels in the codes.  A row with an infinity, a NaN, or a product with its
    weight beyond float32 gets codes 0 and scale NaN.  ``slots`` and ``out`` as in quantize_rows."""
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
    bias[j] (float32 [n]: a prior of each row, or -|x|^2 / 2 for distances).

    The sum over dim is exact.  It is converted to float32 (a rounding beyond 2^24, which takes more than 1,040 values),
    multiplied with the query's scale (a rounding; the product has to stay in the range: values up to 1e32), multiplied
    with the row's and added to the bias in one operation (a rounding), and rounded to ``dtype``.  A
    new result of 256 rows and more starts its rows on 128 bytes (its row stride is n rounded up, so it is only
    contiguous where n allows); ``out`` may have any row stride.  Codes whose rows do not start on 16 bytes or end
    without padding are copied first; those of quantize_rows and Int8Rows never are."""
    return _bind().scores(query_codes, query_scales, codes, scales, bias, dtype, out)


def check_products(device=None) -> None:
    """Waits for the current stream of ``device`` and raises NativeLibraryError if a product on it has given up a
    bounded wait since the last call: int8_scores writes NaN for what it could not compute."""
    with torch.cuda.device(device):
        _native.check(_native.lib().circuit_op_int8_status(torch.cuda.current_stream().cuda_stream), "int8_scores")


def _stream(device: torch.device) -> int:
    """The current stream of a device, as a plain number."""
    return torch._C._cuda_getCurrentRawStream(device.index)


class Int8Rows:
    """A store of 8-bit rows on one device: places that hold a row or none.

    ``codes`` [len, dim] and ``scales`` [len] are what int8_scores and dequantize_rows take; a place without a row has
    scale NaN, reads as NaN and is never a search result.  Calls on one store are ordered by their streams: writing
    places while another stream reads them is the caller's to order.  One thread at a time writes, appends or removes;
    others may read and search meanwhile.  An append that outgrows the buffers moves every
    place to new ones, so to later calls on other streams it counts as writing every place; calls that are under way
    elsewhere still have the old buffers, which are not used again before these calls are done.  ``codes`` and
    ``scales`` taken before an append, and calls captured into a graph before it, see the places as they were then:
    take and capture them again."""

    def __init__(self, places: int, dim: int, device="cuda"):
        if not 1 <= dim <= _native.CIRCUIT_INT8_MAX_DIM or not 0 <= places < 2 ** 31:
            raise ValueError(f"places must be in [0, 2^31) and dim in [1, {_native.CIRCUIT_INT8_MAX_DIM}]")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("8-bit rows live on a CUDA device (no CPU path)")
        self.dim = int(dim)
        self._len = int(places)
        self._in_graph, self._captured = False, []  # a captured call uses the buffers; older buffers of such calls
        codes, scales = self._buffers(self._len)
        self.device = codes.device  # with its index: the current device may change
        self._made = codes, scales, _stream(self.device)  # replaced as a whole: threads that search see one or the other

    def _buffers(self, n: int):
        codes = torch.zeros((n, (self.dim + 15) // 16 * 16), dtype=torch.int8, device=self.device)
        # one scale more than places: what is meant for no place goes there
        return codes, torch.full((n + 1,), float("nan"), dtype=torch.float32, device=self.device)

    def __setstate__(self, state):  # a copy: its buffers are new ones of the current stream, and no graph has them
        self.__dict__.update(state, _in_graph=False, _captured=[])
        self._made = *self._made[:2], _stream(self.device)

    def _use(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Codes and scales for the current stream: their memory is kept for it when a growing store drops them."""
        n, now = self._len, _stream(self.device)  # the length first: later buffers hold as many places
        codes, scales, made_on = self._made
        if now != made_on:
            stream = torch.cuda.current_stream(self.device)
            codes.record_stream(stream)
            scales.record_stream(stream)
        if now and torch.cuda.is_current_stream_capturing():  # never the default stream, 0
            self._in_graph = True
        return codes[:n, :self.dim], scales[:n]

    def __len__(self) -> int:
        return self._len

    @property
    def codes(self) -> torch.Tensor:
        return self._use()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._use()[1]

    def write(self, rows: torch.Tensor, slots: torch.Tensor, normalize: bool = False) -> None:
        """Quantises rows [n, dim] into places slots [n] (int32 or int64).  A slot outside the store writes nothing, of
        equal slots the last row stays."""
        quantize_rows(rows, slots=slots, out=self._use(), normalize=normalize)

    def append(self, rows: torch.Tensor, normalize: bool = False) -> range:
        """Adds rows [n, dim] in new places at the end and returns these places."""
        if not isinstance(rows, torch.Tensor) or rows.ndim != 2 or rows.shape[1] != self.dim:
            raise ValueError("rows must have shape [n, dim]")
        first, need = self._len, self._len + rows.shape[0]
        if need >= 2 ** 31:
            raise ValueError("a store holds less than 2^31 rows")
        self._use()
        codes, scales, _ = self._made
        if need > codes.shape[0]:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a store does not grow inside a graph: each replay would copy the old rows")
            if self._in_graph:
                self._captured.append((codes, scales))
                self._in_graph = False
            old, (codes, scales) = (codes, scales), self._buffers(max(need, 2 * codes.shape[0]))
            codes[:first].copy_(old[0][:first])
            scales[:first].copy_(old[1][:first])
            self._made = codes, scales, _stream(self.device)
        quantize_rows(rows, out=(codes[first:need, :self.dim], scales[first:need]), normalize=normalize)
        self._len = need
        return range(first, need)

    def remove(self, slots: torch.Tensor) -> None:
        """Empties the places ``slots`` (whole numbers, any shape).  A slot outside the store changes nothing."""
        if not isinstance(slots, torch.Tensor) or slots.dtype == torch.bool or slots.is_floating_point() or slots.is_complex():
            raise ValueError("slots must be a tensor of whole numbers")
        self._use()
        codes, scales, _ = self._made
        at = slots.to(device=self.device, dtype=torch.int64).reshape(-1)
        at = at.masked_fill((at < 0) | (at >= self._len), codes.shape[0])
        scales.index_fill_(0, at, float("nan"))

    def read(self, ids: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The rows at ``ids`` (any shape, as a search returns them; -1 gives zeros)."""
        return dequantize_rows(*self._use(), ids, dtype=dtype)

    def scores(self, queries: torch.Tensor, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float32,
               normalize: bool = False) -> torch.Tensor:
        """Products [nq, len] of queries [nq, dim], quantised row by row, with all places."""
        codes, scales = quantize_rows(queries, normalize=normalize)
        return int8_scores(codes, scales, *self._use(), bias=bias, dtype=dtype)

    def search(self, queries: torch.Tensor, k: int = 10, normalize: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
        """The k best places of each query [nq, dim] by its product with the stored rows: (scores [nq, k] descending,
        ids [nq, k] int32), ties to the lower place, score -inf and id -1 where there are fewer rows; 1 <= k <= 256.
        A query with an infinity or NaN has no results.  A place whose row's product is NaN all the same (the kernel
        gave up a wait, see check_products, or left the range of float32) comes first, with score NaN."""
        return self.search_codes(*quantize_rows(queries, normalize=normalize), k=k)

    # scores that are ranked at a time: of so many rows at least, so of so many queries at most
    _BLOCK, _BLOCK_ROWS = 1 << 25, 1 << 14

    def search_codes(self, query_codes: torch.Tensor, query_scales: torch.Tensor, k: int = 10):
        """search with queries that are quantised already."""
        if not 1 <= int(k) <= _native.CIRCUIT_MAX_K:
            raise ValueError(f"k must be in [1, {_native.CIRCUIT_MAX_K}]")
        if (query_codes.ndim != 2 or query_codes.dtype != torch.int8 or query_codes.shape[1] != self.dim or
                query_scales.dtype != torch.float32 or query_scales.shape != query_codes.shape[:1]):
            raise ValueError("queries must be int8 codes [nq, dim] and float32 scales [nq]")
        codes, scales = self._use()
        nq, n = query_codes.shape[0], codes.shape[0]
        most = max(1, self._BLOCK // self._BLOCK_ROWS)
        if nq > most:
            parts = [self.search_codes(query_codes[a:a + most], query_scales[a:a + most], k) for a in range(0, nq, most)]
            return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        none = -(1 << 63)
        best = None
        block = max(self._BLOCK_ROWS, self._BLOCK // max(1, nq))
        for a in range(0, n if nq else 0, block):
            b = min(n, a + block)
            s = int8_scores(query_codes, query_scales, codes[a:b], scales[a:b])
            # one whole number a score: the order of floats (both zeros as 0, NaN above all, as the kernel writes it) in
            # the upper half, the lower place first in the lower half
            order = s.add_(0.0).view(torch.int32)
            order ^= (order >> 31) & 0x7FFFFFFF
            last = 0xFFFFFFFF
            key = torch.add(torch.arange(last - a, last - b, -1, device=self.device), order, alpha=1 << 32)
            key.masked_fill_(scales[a:b].isnan(), none)
            if best is not None:
                key = torch.cat([best, key], 1)
            best = key.topk(min(k, key.shape[1]), dim=1).values
        if best is None or best.shape[1] < k:  # fewer places than results
            more = k - (0 if best is None else best.shape[1])
            blank = torch.full((nq, more), none, dtype=torch.int64, device=self.device)
            best = blank if best is None else torch.cat([best, blank], 1)
        empty = (best == none) | query_scales.isnan()[:, None]
        bits = best >> 32
        bits ^= (bits >> 31) & 0x7FFFFFFF
        scores = bits.to(torch.int32).view(torch.float32).masked_fill_(empty, float("-inf"))
        ids = (~best).to(torch.int32).masked_fill_(empty, -1)  # the lower half
        return scores, ids
