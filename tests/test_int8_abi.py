"""The 8-bit row ops refuse bad arguments on the host, before any CUDA call, and leave the reason behind."""
import ctypes

import numpy as np
import pytest
import torch

from circuit_rag import _native
from circuit_rag.int8 import dequantize_rows, int8_scores, quantize_rows, rms_norm_quantize

ARG = -2
# 16-byte aligned host memory: never read, every call below is refused or has nothing to do
_BUF = np.zeros(4096 + 16, np.uint8)
P = (_BUF.ctypes.data + 15) // 16 * 16


def quantize(rows=P, dtype=0, n=2, dim=8, stride=8, res=None, res_stride=8, w=None, w_dtype=0, norm=0, eps=0.0,
             summed=None, sum_stride=8, slots=None, slot_bytes=0, cap=2, codes=P, code_stride=16, scales=P):
    return _native.lib().circuit_op_quantize_rows(rows, dtype, n, dim, stride, res, res_stride, w, w_dtype, norm, eps,
                                                  summed, sum_stride, slots, slot_bytes, cap, codes, code_stride,
                                                  scales, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(dim=0), dict(dim=16385, stride=20000, code_stride=20000), dict(n=-1),
    dict(n=1 << 31, cap=1 << 32), dict(norm=3), dict(norm=-1), dict(w=P), dict(res=P, summed=P), dict(norm=1, res=P),
    dict(norm=1, eps=-1.0), dict(norm=1, eps=float("nan")), dict(norm=1, eps=float("inf")),
    dict(norm=1, w=P, w_dtype=1), dict(dtype=2, norm=1, w=P, w_dtype=1), dict(slots=P, slot_bytes=2), dict(cap=-1),
    dict(rows=None), dict(codes=None), dict(scales=None), dict(cap=1), dict(stride=7), dict(code_stride=7),
    dict(norm=1, res=P, summed=P, res_stride=7), dict(norm=1, res=P, summed=P, sum_stride=7), dict(rows=P + 2),
    dict(dtype=1, rows=P + 1), dict(norm=1, res=P + 1, summed=P), dict(norm=1, res=P, summed=P + 2),
    dict(norm=1, w=P + 2), dict(slots=P + 2, slot_bytes=4), dict(slots=P + 4, slot_bytes=8), dict(scales=P + 1)])
def test_quantize_refuses(bad):
    assert quantize(**bad) == ARG
    assert "quantize_rows" in _native.last_error()


def test_quantize_of_nothing():
    assert quantize(n=0, rows=None, codes=None, scales=None, cap=0) == 0


def dequantize(codes=P, code_stride=16, scales=P, rows=4, dim=8, ids=None, id_bytes=0, n=4, out=P, dtype=0,
               out_stride=8):
    return _native.lib().circuit_op_dequantize_rows(codes, code_stride, scales, rows, dim, ids, id_bytes, n, out,
                                                    dtype, out_stride, None)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(dim=0), dict(dim=16385, code_stride=20000, out_stride=20000),
                                 dict(n=-1), dict(n=1 << 31), dict(rows=-1), dict(ids=P, id_bytes=3),
                                 dict(codes=None), dict(scales=None), dict(out=None), dict(n=5), dict(code_stride=7),
                                 dict(out_stride=7), dict(out=P + 2), dict(ids=P + 4, id_bytes=8), dict(scales=P + 2)])
def test_dequantize_refuses(bad):
    assert dequantize(**bad) == ARG
    assert "dequantize_rows" in _native.last_error()


def scores(q=P, q_stride=16, qs=P, nq=2, codes=P, code_stride=16, s=P, n=4, dim=8, bias=None, out=P, dtype=0,
           out_stride=4):
    return _native.lib().circuit_op_int8_scores(q, q_stride, qs, nq, codes, code_stride, s, n, dim, bias, out, dtype,
                                                out_stride, None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dim=0), dict(dim=16385, q_stride=20000, code_stride=20000),
                                 dict(nq=-1), dict(nq=65536), dict(n=-1), dict(n=1 << 31, out_stride=1 << 31),
                                 dict(q=None), dict(qs=None), dict(codes=None), dict(s=None), dict(out=None),
                                 dict(q_stride=8), dict(code_stride=8), dict(q_stride=24), dict(code_stride=24),
                                 dict(dim=17), dict(q=P + 8), dict(codes=P + 1), dict(out_stride=3), dict(out=P + 2),
                                 dict(qs=P + 2), dict(s=P + 1), dict(bias=P + 2)])
def test_scores_refuses(bad):
    assert scores(**bad) == ARG
    assert "int8_scores" in _native.last_error()


def test_nothing_to_do():
    assert dequantize(n=0, out=None) == 0
    assert scores(nq=0) == 0 and scores(n=0, out_stride=0) == 0


def test_python_refuses_cpu_tensors():
    x = torch.randn(2, 16)
    c, s = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: quantize_rows(x), lambda: rms_norm_quantize(x), lambda: dequantize_rows(c, s),
                 lambda: int8_scores(c, s, c, s), lambda: quantize_rows(None)):
        with pytest.raises(RuntimeError):
            call()


def test_symbols_have_signatures():
    for name in ("circuit_op_quantize_rows", "circuit_op_dequantize_rows", "circuit_op_int8_scores"):
        assert getattr(_native.lib(), name).restype is ctypes.c_int


def test_rag_refuses_8_bit_rows_on_the_cpu():
    from circuit_rag import CircuitRAG

    with pytest.raises(ValueError):
        CircuitRAG(device="cpu", embed_fn=len, rows="int4")
    rag = CircuitRAG(device="cpu", embed_fn=lambda texts: np.ones((len(texts), 4), np.float32), rows="int8")
    with pytest.raises(RuntimeError):
        rag.add_documents(["a"])
    assert rag.texts == [] and rag.search("a") == []
    with pytest.raises(ValueError):
        CircuitRAG(device="cpu", embed_fn=len).search("a", feedback=[1])
