"""8-bit rows on the GPU (quantise, norm, write, read, products) against the formulas in 64 bits.

Tolerances.  Codes are the correctly rounded quotients: equal.  A plain scale is one fp32 division: equal.  A norm's
scale has four more roundings and the fp32 sum of squares (at most 64 terms a thread in a row, then a tree of 9 levels;
the error halves under the root): (4 + (64 + 9 + 1) / 2) 2^-24 < 2.5e-6 relative.  A read value is one fp32 product and
one rounding to its type; a score three fp32 roundings and one to its type (a rounding: eps / 2)."""
import math
import os
import subprocess
import sys

import pytest
import torch

from circuit_rag import _native
from circuit_rag.int8 import dequantize_rows, int8_scores, quantize_rows, rms_norm_quantize

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NORM_SCALE_RTOL = 2.5e-6
U32 = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _rows(n, d, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(n, d, generator=g, device=DEV) * scale).to(dtype)


def _want(u):
    """Codes and max|u| of the rows of u (64 bits)."""
    a = u.abs().amax(1)
    c = torch.round(u * 127.0 / torch.where(a > 0, a, 1)[:, None])
    return c.to(torch.int8), a


def _check_plain(x, codes, scales):
    c, a = _want(x.double())
    assert torch.equal(codes, c)
    assert torch.equal(scales, (a / 127).float())


DIMS = [1, 2, 6, 7, 16, 31, 33, 64, 100, 128, 130, 136, 200, 256, 384, 385, 511, 512, 513, 514, 604, 640, 768, 1000, 1024,
        1025, 1030, 1536, 2048, 2049, 4096, 4100, 4102, 8191, 8192, 8196, 8198, 16382, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", DIMS)
def test_quantize_dims(d, dtype):
    for n in (1, 5, 67, 701, 1300):
        x = _rows(n, d, dtype, seed=d + n)
        codes, scales = quantize_rows(x)
        assert codes.shape == (n, d) and codes.dtype == torch.int8 and scales.dtype == torch.float32
        _check_plain(x, codes, scales)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strides_and_alignment(dtype):
    big = _rows(40, 700, dtype, seed=3)
    for x in (big[:, :384], big[:, 1:385], big[:, 3:388], big[::3, 8:392], big.T, big[:, ::2], big[5:6, 2:99],
              big[0].expand(9, 700)):
        codes, scales = quantize_rows(x)
        _check_plain(x, codes, scales)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_ties_go_to_even(dtype):
    # maxima of 127 times a power of two: every second value is a half; others: only top / 2 is
    x = torch.arange(-127, 128, device=DEV).repeat_interleave(2)[:504].float() / 2
    x[-1] = 127.0
    rows = torch.stack([x, x * 2.0 ** -7, -x, x / 2 ** 6]).to(dtype)
    top = torch.tensor([1.0, 1.25, 127.0, 254.0, 190.5, 1.9921875, 3.0, 0.0078125], device=DEV)[:, None]
    half = torch.cat([top, top / 2, -top / 2, top / 4, -top, torch.zeros_like(top), top / 2, top * 0.75], 1).to(dtype)
    for y in (rows, rows.repeat(200, 1), half, half.repeat(300, 7), half.float(), torch.cat([half, half[:, :1]], 1)):
        codes, scales = quantize_rows(y)
        _check_plain(y, codes, scales)
        codes, scales = quantize_rows(y, normalize=True)
        _check_norm(y, None, None, 0.0, (codes, scales, None), unit=True)
    # 16-bit rows of every significand of the maximum
    g = torch.Generator(device=DEV).manual_seed(1)
    bits = torch.arange(0, 2 ** 11, device=DEV)
    top = (1 + bits / 2 ** 11).to(dtype)[:, None]
    y = torch.cat([top, (torch.rand(2048, 255, generator=g, device=DEV) * top).to(dtype)], 1)
    _check_plain(y, *quantize_rows(y))


def test_quantize_next_to_halves():
    # values one step of fp32 around (k + 1/2) a / 127 for odd a: only the exact quotient tells the code
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        a = torch.rand(1, generator=g).double() + 0.5
        a = a.float().double()
        k = torch.arange(-126, 126).double() + 0.5
        mid = (k * a / 127).float()
        x = torch.cat([a.float(), mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)])[None].to(DEV)
        codes, scales = quantize_rows(x)
        _check_plain(x, codes, scales)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-44, 1e-40, 1e-38, 1e-30, 1e-18, 1e30, 1e36, 1e37])
def test_quantize_extreme_magnitudes(scale, dtype):
    x = _rows(6, 260, torch.float32, seed=1)
    x = (x.double() * scale).to(dtype)
    for y in (x, x[:, 1:], x.repeat(120, 1)):
        codes, scales = quantize_rows(y)
        _check_plain(y, codes, scales)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [5, 384, 3000, 9000])
def test_zero_and_not_finite_rows(d, dtype):
    x = _rows(8, d, dtype, seed=2)
    x[1] = 0
    x[2, d // 2] = float("nan")
    x[3, 0] = float("inf")
    x[4, d - 1] = -float("inf")
    x[5] = -0.0
    good = [0, 1, 5, 6, 7]
    codes, scales = quantize_rows(x)
    _check_plain(x[good], codes[good], scales[good])
    assert (codes[2:5] == 0).all() and scales[2:5].isnan().all()
    assert scales[1] == 0 and scales[5] == 0
    back = dequantize_rows(codes, scales, dtype=dtype)
    assert back[2:5].isnan().all() and (back[1] == 0).all()
    codes, scales, _ = rms_norm_quantize(x, eps=0.0)
    assert scales[2:5].isnan().all() and (codes[2:5] == 0).all() and scales[1] == 0 and scales[5] == 0


def _check_norm(x, r, w, eps, got, unit=False):
    codes, scales, summed = got
    if r is None:
        v = x.double()
        assert summed is None
    else:
        v = (x.float() + r.float()).to(x.dtype).double()
        assert torch.equal(summed.double(), v)
    u = v if w is None else v * w.double()
    c, a = _want(u)
    assert torch.equal(codes, c)
    ss = v.square().sum(1) if unit else v.square().mean(1)
    want = a / 127 / torch.sqrt(ss + eps)
    want = torch.where(a == 0, 0, want)
    torch.testing.assert_close(scales.double(), want, rtol=NORM_SCALE_RTOL, atol=2.0 ** -149)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", DIMS)
def test_norm_dims(d, dtype):
    for n in (1, 37, 613, 1250):
        x, r = _rows(n, d, dtype, seed=d), _rows(n, d, dtype, seed=d + 1, scale=0.3)
        w = (1 + 0.2 * _rows(1, d, torch.float32, seed=d + 2)[0])
        for rr, ww in ((r, w.to(dtype)), (r, w), (None, w), (r, None), (None, None)):
            _check_norm(x, rr, ww, 1e-6, rms_norm_quantize(x, residual=rr, weight=ww))
        codes, scales = quantize_rows(x, normalize=True)
        _check_norm(x, None, None, 0.0, (codes, scales, None), unit=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_strides(dtype):
    big, other, w = _rows(30, 900, dtype, seed=4), _rows(30, 800, dtype, seed=5), _rows(2, 900, dtype, seed=6)
    for x, r in ((big[:, :511], other[:, 1:512]), (big[:, 3:515], other[:, :512]), (big.T[:30, :30], other[:, 8:38])):
        for ww in (w[0, :x.shape[1]], w[1, 1:1 + x.shape[1]], w.T.reshape(-1)[:2 * x.shape[1]:2]):
            _check_norm(x, r, ww, 1e-5, rms_norm_quantize(x, residual=r, weight=ww, eps=1e-5))


@pytest.mark.parametrize("scale", [1e-40, 1e-30, 1e-22, 1e-15, 1e15, 1e19, 1e25, 1e37])
@pytest.mark.parametrize("d", [384, 6000])
def test_norm_extreme_magnitudes(scale, d):
    x = (_rows(5, d, torch.float32, seed=7).double() * scale).float()
    mixed = torch.cat([x, _rows(5, d, torch.float32, seed=8)]).repeat(80, 1)  # rows in and out of range in one warp
    for y in (x, x[:, 1:], mixed):
        _check_norm(y, None, None, 0.0, rms_norm_quantize(y, eps=0.0))
        _check_norm(y, None, None, 1e-6, rms_norm_quantize(y, eps=1e-6))


def test_norm_sum_overflows_its_type():
    x = torch.full((2, 64), 60000.0, dtype=torch.float16, device=DEV)
    x[1] = 1.0
    codes, scales, summed = rms_norm_quantize(x, residual=x)
    assert summed[0].isinf().all() and scales[0].isnan() and (codes[0] == 0).all()
    _check_norm(x[1:], x[1:], None, 1e-6, (codes[1:], scales[1:], summed[1:]))


def _store(cap, d, fill=77):
    buf = torch.full((cap, (d + 15) // 16 * 16), fill, dtype=torch.int8, device=DEV)
    return buf, buf[:, :d], torch.full((cap,), -3.5, device=DEV)


@pytest.mark.parametrize("sdtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [1, 2, 40, 1024, 1025, 5000])
@pytest.mark.parametrize("d", [9, 384, 5000])
def test_write_to_slots(n, d, sdtype):
    cap = n + 50
    dtype = TYPES[n % 3]
    x = _rows(n, d, dtype, seed=n)
    g = torch.Generator().manual_seed(n)
    # many equal slots, empty places and slots past the end
    slots = torch.randint(-3, cap + 4, (n,), generator=g)
    slots[n // 2:] = slots[:n - n // 2].clone()
    buf, codes, scales = _store(cap, d)
    out = quantize_rows(x, slots=slots.to(DEV, sdtype), out=(codes, scales))
    assert out[0].data_ptr() == codes.data_ptr() and out[1].data_ptr() == scales.data_ptr()
    c, a = _want(x.double())
    want_b, want_c, want_s = _store(cap, d)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < cap:
            want_c[s] = c[i]
            want_s[s] = (a[i] / 127).float()
    assert torch.equal(buf, want_b)
    assert torch.equal(scales, want_s)


@pytest.mark.parametrize("n", [30, 3000])
def test_write_every_row_to_one_slot(n):
    x = _rows(n, 128, torch.float32, seed=n)
    buf, codes, scales = _store(4, 128)
    codes2, scales2, summed = rms_norm_quantize(x, residual=x, slots=torch.full((n,), 2, device=DEV),
                                                out=(codes, scales))
    _check_norm(x[-1:], x[-1:], None, 1e-6, (codes[2:3], scales[2:3], summed[-1:]))
    assert torch.equal(summed, x + x)  # the rows that were not kept are summed all the same
    for i in (0, 1, 3):
        assert (codes[i] == 77).all() and scales[i] == -3.5


def test_write_nothing():
    buf, codes, scales = _store(4, 32)
    x = _rows(3, 32, torch.float32)
    quantize_rows(x, slots=torch.tensor([-1, 4, 1 << 40], device=DEV), out=(codes, scales))
    quantize_rows(x[:0], slots=torch.empty(0, dtype=torch.int64, device=DEV), out=(codes, scales))
    assert (codes == 77).all() and (scales == -3.5).all()
    empty = quantize_rows(x[:0])
    assert empty[0].shape == (0, 32) and empty[1].shape == (0,)
    x2 = x.half()
    _, _, summed = rms_norm_quantize(x2, residual=x2, slots=torch.tensor([-1, 0, 3], device=DEV),
                                     out=(codes[:0], scales[:0]))
    assert torch.equal(summed, x2 + x2)


def test_write_into_unpadded_codes():
    for d in (384, 37, 20):
        x = _rows(9, d, torch.bfloat16, seed=d)
        flat = torch.full((9 * d + 3,), 5, dtype=torch.int8, device=DEV)
        codes, scales = flat[3:].view(9, d), torch.empty(9, device=DEV)
        quantize_rows(x, out=(codes, scales))
        _check_plain(x, codes, scales)
        assert (flat[:3] == 5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 5, 16, 100, 384, 1000, 4099])
def test_read(d, dtype):
    x = _rows(300, d, torch.float32, seed=d, scale=3.0)
    codes, scales = quantize_rows(x)
    want = (codes.double() * scales.double()[:, None])
    tol = U32 + _half(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    got = dequantize_rows(codes, scales, dtype=dtype)
    assert got.dtype == dtype
    assert ((got.double() - want).abs() <= tol * (1 + tol) * want.abs() + tiny).all()
    ids = torch.tensor([[3, -1, 299], [0, 3, 300]], device=DEV, dtype=torch.int32)
    for i in (ids, ids.long(), ids.T):
        got_i = dequantize_rows(codes, scales, i, dtype=dtype)
        assert got_i.shape == (*i.shape, d)
        for at, row in zip(i.reshape(-1).tolist(), got_i.reshape(-1, d)):
            if at == 300:
                assert row.isnan().all()
            else:
                assert torch.equal(row, got[at] if at >= 0 else torch.zeros_like(row))
    wide = torch.full((3, d + 9), 2.0, dtype=dtype, device=DEV)
    dequantize_rows(codes, scales, ids[0], dtype=dtype, out=wide[:, 3:3 + d])
    assert torch.equal(wide[:, 3:3 + d], torch.stack([got[3], torch.zeros_like(got[3]), got[299]]))
    assert (wide[:, :3] == 2).all() and (wide[:, 3 + d:] == 2).all()
    assert dequantize_rows(codes, scales, ids[:0], dtype=dtype).shape == (0, 3, d)
    flat = torch.cat([codes[0, :1], codes.reshape(-1)])  # rows that start anywhere
    assert torch.equal(dequantize_rows(flat[1:].view(300, d), scales, dtype=dtype), got)


def _scores_want(qc, qs, rc, rs, bias):
    acc = (qc.double() @ rc.double().T)
    prod = acc * qs.double()[:, None] * rs.double()[None]
    return prod, prod if bias is None else prod + bias.double()[None]


def _check_scores(got, qc, qs, rc, rs, bias, dtype):
    prod, want = _scores_want(qc, qs, rc, rs, bias)
    tol = 3 * U32 * (prod.abs() + (0 if bias is None else bias.double().abs()[None]))
    tol = tol + _half(dtype) * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert got.dtype == dtype and got.shape == want.shape
    off = (got.double() - want).abs() > tol
    assert not off.any(), (int(off.sum()), off.nonzero()[:5].tolist())


def _codes(n, d, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c = torch.randint(-127, 128, (n, (d + 15) // 16 * 16), generator=g, device=DEV, dtype=torch.int8)
    s = torch.rand(n, generator=g, device=DEV) * 0.01 + 1e-4
    return c[:, :d], s  # the padding holds codes too: it must not count


@pytest.mark.parametrize("d", [1, 15, 16, 17, 33, 100, 128, 129, 384, 400, 1000, 2048, 5000, 16384])
@pytest.mark.parametrize("nq,n", [(1, 1), (1, 1000), (2, 33), (3, 257), (4, 128), (7, 31), (8, 300), (9, 129), (16, 1000),
                                  (33, 513), (129, 127), (300, 700)])
def test_scores_sizes(nq, n, d):
    qc, qs = _codes(nq, d, seed=d + nq)
    rc, rs = _codes(n, d, seed=d + n + 7)
    dtype = TYPES[(nq + n + d) % 3]
    bias = torch.randn(n, device=DEV) if (nq + d) % 2 else None
    _check_scores(int8_scores(qc, qs, rc, rs, bias=bias, dtype=dtype), qc, qs, rc, rs, bias, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq", [1, 6, 64, 257])
def test_scores_types_strides_and_out(nq, dtype):
    qc, qs = _codes(nq, 200, seed=nq)
    rc, rs = _codes(1003, 200, seed=nq + 1)
    bias = torch.randn(1003, device=DEV)
    wide = torch.full((nq + 2, 1003 + 21), 9.0, dtype=dtype, device=DEV)
    out = wide[1:-1, 5:1008]
    got = int8_scores(qc, qs, rc, rs, bias=bias, dtype=dtype, out=out)
    assert got.data_ptr() == out.data_ptr()
    _check_scores(got, qc, qs, rc, rs, bias, dtype)
    rest = wide.clone()
    rest[1:-1, 5:1008] = 9.0
    assert (rest == 9.0).all()  # nothing around the result is written
    want = got.clone()
    # rows that do not start on 16 bytes, unpadded rows, transposed codes, every second row
    flat = torch.empty(1003 * 200 + 1, dtype=torch.int8, device=DEV)
    flat[1:] = rc.reshape(-1)
    both = torch.stack([rc, rc], 1).reshape(2006, 200)
    for r in (flat[1:].view(1003, 200), rc.contiguous(), rc.T.contiguous().T, both[::2]):
        assert torch.equal(int8_scores(qc, qs, r, rs, bias=bias, dtype=dtype), want)
    scattered = torch.stack([rs, rs], 1)[:, 0]
    assert torch.equal(int8_scores(qc, qs, rc, scattered, bias=bias, dtype=dtype), want)


@pytest.mark.parametrize("nq", [1, 5, 40, 200])
def test_scores_extreme_codes(nq):
    d = 16384
    qc = torch.full((nq, d), -128, dtype=torch.int8, device=DEV)
    rc = torch.full((130, d), -128, dtype=torch.int8, device=DEV)
    rc[1::2] = 127
    one = torch.ones(200, device=DEV)
    got = int8_scores(qc, one[:nq], rc, one[:130])
    assert (got[:, 0::2] == float(128 * 128 * d)).all() and (got[:, 1::2] == float(-128 * 127 * d)).all()


@pytest.mark.parametrize("nq", [1, 3, 70])
def test_scores_of_empty_and_bad_rows(nq):
    qc, qs = _codes(nq, 64, seed=1)
    rc, rs = _codes(200, 64, seed=2)
    rs[5], rs[6] = 0.0, float("nan")
    rc[6] = 0
    got = int8_scores(qc, qs, rc, rs)
    assert (got[:, 5] == 0).all() and got[:, 6].isnan().all() and not got[:, 7:].isnan().any()
    assert int8_scores(qc[:0], qs[:0], rc, rs).shape == (0, 200)
    assert int8_scores(qc, qs, rc[:0], rs[:0]).shape == (nq, 0)


@pytest.mark.parametrize("nq", [2, 17])
def test_scores_past_32_bits(nq):
    # codes of more than 2^32 bytes: rows on both sides of the border
    d, n = 16384, (1 << 18) + 300
    rc = torch.zeros(n, d, dtype=torch.int8, device=DEV)
    rs = torch.ones(n, device=DEV)
    marks = torch.tensor([0, 131071, 131072, 262143, 262144, n - 1], device=DEV)
    some, _ = _codes(len(marks), d, seed=3)
    rc[marks] = some
    qc, qs = _codes(nq, d, seed=4)
    got = int8_scores(qc, qs, rc, rs)
    _check_scores(got[:, marks], qc, qs, some, rs[marks], None, torch.float32)
    got[:, marks] = 0
    assert (got == 0).all()
    back = dequantize_rows(rc, rs, marks)
    assert torch.equal(back, some.float())
    new = _rows(2, d, torch.float32)
    quantize_rows(new, slots=torch.tensor([262143, 262144 + 7], device=DEV), out=(rc, rs))
    _check_plain(new, rc[[262143, 262151]], rs[[262143, 262151]])


def test_scores_result_past_32_bits():
    nq, n = 4200, 520_000  # 2.18e9 results
    qc, qs = _codes(nq, 16, seed=1)
    rc, rs = _codes(n, 16, seed=2)
    got = int8_scores(qc, qs, rc, rs, dtype=torch.bfloat16)
    for a, b in ((0, 0), (nq - 5, n - 300), (4130, 1000)):
        _check_scores(got[a:a + 5, b:b + 300], qc[a:a + 5], qs[a:a + 5], rc[b:b + 300], rs[b:b + 300], None,
                      torch.bfloat16)


def test_refusals():
    x = _rows(4, 32, torch.float32)
    codes, scales = quantize_rows(x)
    cpu = x.cpu()
    for call in (lambda: quantize_rows(cpu), lambda: rms_norm_quantize(x, residual=cpu),
                 lambda: dequantize_rows(codes.cpu(), scales), lambda: int8_scores(codes, scales, codes.cpu(), scales),
                 lambda: quantize_rows(x.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: quantize_rows(x.double()), lambda: quantize_rows(x[0]), lambda: quantize_rows(x.int()),
                 lambda: quantize_rows(x, slots=torch.zeros(4, device=DEV, dtype=torch.int64)),
                 lambda: quantize_rows(x, slots=torch.zeros(3, device=DEV, dtype=torch.int64), out=(codes, scales)),
                 lambda: quantize_rows(x, slots=torch.zeros(4, device=DEV), out=(codes, scales)),
                 lambda: quantize_rows(x[:3], out=(codes, scales)), lambda: quantize_rows(x[:, :16], out=(codes, scales)),
                 lambda: quantize_rows(x, out=(codes[:1].expand(4, 32), scales)),
                 lambda: quantize_rows(x, out=(codes, scales[:1].expand(4))),
                 lambda: quantize_rows(torch.zeros(1, 16385, device=DEV)), lambda: quantize_rows(x[:, :0]),
                 lambda: rms_norm_quantize(x, residual=x[:3]), lambda: rms_norm_quantize(x, residual=x.half()),
                 lambda: rms_norm_quantize(x, weight=x), lambda: rms_norm_quantize(x, weight=x[0].half()),
                 lambda: rms_norm_quantize(x, eps=-1.0), lambda: rms_norm_quantize(x, eps=math.nan),
                 lambda: dequantize_rows(codes, scales, torch.zeros(2, device=DEV)),
                 lambda: dequantize_rows(codes, scales, dtype=torch.float64),
                 lambda: dequantize_rows(codes, scales[:3]), lambda: dequantize_rows(codes.float(), scales),
                 lambda: dequantize_rows(codes, scales, out=torch.empty(3, 32, device=DEV)),
                 lambda: int8_scores(codes, scales, codes[:, :16], scales),
                 lambda: int8_scores(codes, scales, codes, scales, bias=torch.zeros(3, device=DEV)),
                 lambda: int8_scores(codes, scales, codes, scales, dtype=torch.int32),
                 lambda: int8_scores(codes, scales, codes, scales, out=torch.empty(4, 5, device=DEV))):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        quantize_rows(x.clone().requires_grad_())


@pytest.mark.parametrize("nq", [1, 40, 300])
def test_together_on_a_side_stream_and_in_a_graph(nq):
    """Norm, write, read and products one after the other, as a program runs them: eager on a side stream, then
    captured once and replayed on new inputs."""
    d, cap = 384, 3000
    x, r, w = _rows(500, d, torch.bfloat16, 1), _rows(500, d, torch.bfloat16, 2), _rows(1, d, torch.bfloat16, 3)[0]
    slots = torch.randperm(cap, device=DEV)[:500]
    q = _rows(nq, d, torch.float32, 4)
    buf, codes, scales = _store(cap, d, fill=0)
    scales.zero_()

    def step():
        rms_norm_quantize(x, residual=r, weight=w, slots=slots, out=(codes, scales))
        back = dequantize_rows(codes, scales, slots)
        qc, qs = quantize_rows(q)
        return back, qc, qs, int8_scores(qc, qs, codes, scales)

    def check(got):
        back, qc, qs, s = got
        v = (x.float() + r.float()).to(torch.bfloat16).double()
        c, a = _want(v * w.double())
        assert torch.equal(codes[slots], c)
        assert torch.equal(back, codes[slots].float() * scales[slots][:, None])
        _check_plain(q, qc, qs)
        _check_scores(s, qc, qs, codes, scales, None, torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    check(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (10, 20):
        x.copy_(_rows(500, d, torch.bfloat16, seed))
        q.copy_(_rows(nq, d, torch.float32, seed + 1))
        graph.replay()
        torch.cuda.synchronize()
        check(got)


def test_no_wait_has_given_up():
    assert _native.lib().circuit_op_int8_status(None) == 0


def test_layout_of_new_results():
    qc, qs = _codes(5, 64, seed=1)
    for n in (1, 255, 256, 300, 1000):
        rc, rs = _codes(n, 64, seed=n)
        for dtype in TYPES:
            got = int8_scores(qc, qs, rc, rs, dtype=dtype)
            _check_scores(got, qc, qs, rc, rs, None, dtype)
            line = 128 // got.element_size()
            assert got.stride() == (n if n < 256 else -(-n // line) * line, 1)
    one = int8_scores(qc[:1], qs[:1], rc, rs)
    assert one.is_contiguous() and one.shape == (1, 1000)


def test_gradients_are_refused_everywhere():
    x = _rows(4, 32, torch.float32)
    codes, scales = quantize_rows(x)
    wants = [t.clone().requires_grad_() for t in (x, x[0], scales)]
    for call in (lambda: rms_norm_quantize(wants[0]), lambda: rms_norm_quantize(x, residual=wants[0]),
                 lambda: rms_norm_quantize(x, weight=wants[1]), lambda: dequantize_rows(codes, wants[2]),
                 lambda: int8_scores(codes, wants[2], codes, scales), lambda: int8_scores(codes, scales, codes, wants[2]),
                 lambda: int8_scores(codes, scales, codes, scales, bias=wants[2]),
                 lambda: quantize_rows(x, out=(codes, wants[2]))):
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        int8_scores(codes, wants[2], codes, scales)


def test_calls_of_two_streams_at_once():
    """Products and writes of two stores on two streams, each as if it were alone."""
    work = []
    for seed in (1, 2):
        x = _rows(3000, 512, torch.bfloat16, seed)
        rc, rs = _codes(40000, 512, seed + 10)
        qc, qs = _codes(200, 512, seed + 20)
        _, codes, scales = _store(5000, 512, 0)
        work.append((x, rc, rs, qc, qs, codes, scales, torch.randperm(5000, device=DEV)[:3000]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(5):
        for k, (x, rc, rs, qc, qs, codes, scales, slots) in enumerate(work):
            with torch.cuda.stream(streams[k]):
                quantize_rows(x, slots=slots, out=(codes, scales))
                got[k].append(int8_scores(qc, qs, rc, rs))
    torch.cuda.synchronize()
    for k, (x, rc, rs, qc, qs, codes, scales, slots) in enumerate(work):
        _check_plain(x, codes[slots], scales[slots])
        for s in got[k]:
            assert torch.equal(s, got[k][0])
        _check_scores(got[k][0], qc, qs, rc, rs, None, torch.float32)


def test_norm_in_place_of_its_inputs():
    """The C entry's sum may be the rows or the residual themselves."""
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        for d in (384, 385, 5000):
            x, r, w = _rows(70, d, dtype, 1), _rows(70, d, dtype, 2), _rows(1, d, dtype, 3)[0]
            x[5] *= 1e-30 if dtype == torch.float32 else 1
            r[5] *= 1e-30 if dtype == torch.float32 else 1
            for into in (0, 1):
                pair = [x.clone(), r.clone()]
                codes, scales = torch.empty(70, d + 3, dtype=torch.int8, device=DEV)[:, :d], torch.empty(70, device=DEV)
                rc = _native.lib().circuit_op_quantize_rows(
                    pair[0].data_ptr(), code, 70, d, d, pair[1].data_ptr(), d, w.data_ptr(), code, 1, 1e-6,
                    pair[into].data_ptr(), d, None, 0, 70, codes.data_ptr(), d + 3, scales.data_ptr(),
                    torch.cuda.current_stream().cuda_stream)
                assert rc == 0
                _check_norm(x, r, w, float(torch.tensor(1e-6)), (codes, scales, pair[into]))


@pytest.mark.parametrize("d", [20, 130, 384, 1000, 2500])
@pytest.mark.parametrize("nq", [1, 3, 16, 17, 40, 64, 100, 128, 129, 256, 300, 500, 1000])
def test_scores_of_many_rows(nq, d):
    """Several row tiles a block, full and partial ones, in every kernel: the queries' tile kept, streamed, or paired."""
    n = 60001
    dtype = TYPES[(nq + d) % 3]
    qc, qs = _codes(nq, d, seed=d + nq)
    rc, rs = _codes(n, d, seed=d)
    bias = torch.randn(n, device=DEV) if nq % 2 else None
    out = None if d % 20 else torch.empty(nq, n, dtype=dtype, device=DEV)  # rows off 128 bytes
    _check_scores(int8_scores(qc, qs, rc, rs, bias=bias, dtype=dtype, out=out), qc, qs, rc, rs, bias, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [3, 16, 24, 33, 64, 100, 130, 384, 385, 514, 1000, 1030, 1100, 2500, 8200])
def test_read_many_rows(d, dtype):
    codes, scales = _codes(1500, d, seed=d)
    ids = torch.randint(-1, 1500, (3000,), device=DEV)
    want = torch.where((ids >= 0)[:, None], codes[ids].double() * scales[ids].double()[:, None], 0)
    tol = U32 + _half(dtype)
    for rows in (codes, codes.contiguous()):
        got = dequantize_rows(rows, scales, ids, dtype=dtype)
        assert ((got.double() - want).abs() <= tol * (1 + tol) * want.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("n", [700, 4000])
@pytest.mark.parametrize("d", [24, 384, 385, 5000])
def test_write_at_unit_length(n, d):
    x = _rows(n, d, torch.float16, seed=d)
    slots = torch.randint(0, n, (n,), generator=torch.Generator().manual_seed(1))
    buf, codes, scales = _store(n, d)
    quantize_rows(x, slots=slots.to(DEV), out=(codes, scales), normalize=True)
    last = {s: i for i, s in enumerate(slots.tolist())}
    at, row = torch.tensor(list(last), device=DEV), torch.tensor(list(last.values()), device=DEV)
    _check_norm(x[row], None, None, 0.0, (codes[at], scales[at], None), unit=True)
    left = torch.ones(n, dtype=torch.bool, device=DEV)
    left[at] = False
    assert (codes[left] == 77).all() and (scales[left] == -3.5).all()


def test_first_calls_inside_a_capture():
    """Nothing of the calls needs an eager one first: a fresh process captures them at once."""
    code = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from circuit_rag.int8 import dequantize_rows, int8_scores, quantize_rows, rms_norm_quantize
x, y = torch.randn(4000, 256, device="cuda"), torch.randn(300, 256, device="cuda")
slots = torch.randperm(4000, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a = quantize_rows(x)
    b = rms_norm_quantize(y, residual=y)
    quantize_rows(x, slots=slots, out=a)
    results = [int8_scores(b[0][:n], b[1][:n], *a) for n in (1, 16, 64, 128, 300)]
    back = dequantize_rows(*a, slots)
graph.replay()
torch.cuda.synchronize()
for r, n in zip(results, (1, 16, 64, 128, 300)):
    want = (b[0][:n].double() @ a[0].double().T) * b[1][:n, None].double() * a[1].double()
    torch.testing.assert_close(r.double(), want, rtol=1e-6, atol=0)
assert torch.equal(back, a[0][slots].float() * a[1][slots][:, None])
print("captured")
"""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "circuit-rag_b200")
    done = subprocess.run([sys.executable, "-c", code, root], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("d", [1, 16, 33, 64, 100, 128])
@pytest.mark.parametrize("nq", [3, 16, 30, 32, 57, 64])
def test_scores_of_many_short_rows(nq, d):
    """Rows of one chunk, two tiles of them at a time, the last one partial."""
    for n in (200_001, 300_160, 152_000 + 130):
        dtype = TYPES[(nq + d + n) % 3]
        qc, qs = _codes(nq, d, seed=d + nq)
        rc, rs = _codes(n, d, seed=d)
        bias = torch.randn(n, device=DEV) if nq % 2 else None
        _check_scores(int8_scores(qc, qs, rc, rs, bias=bias, dtype=dtype), qc, qs, rc, rs, bias, dtype)


@pytest.mark.parametrize("nq,n", [(1, 3000), (2, 60000), (40, 9000), (300, 9000), (1000, 40000)])
def test_chains_over_the_same_buffers(nq, n):
    """Kernels of a chain start early and wait for the one before: the same buffers are written and read again and
    again without a synchronisation, and every step's results are those of its own inputs."""
    d = 256
    rc, rs = _codes(n, d, seed=n)
    inputs = [_rows(nq, d, torch.bfloat16, seed) for seed in range(6)]
    x = torch.empty_like(inputs[0])
    qc, qs = torch.empty(nq, d, dtype=torch.int8, device=DEV), torch.empty(nq, device=DEV)
    out, back = torch.empty(nq, n, device=DEV), torch.empty(nq, d, device=DEV)
    slots = torch.randperm(n, device=DEV)[:nq]
    kept = []
    torch.cuda.synchronize()
    for step in range(24):
        x.copy_(inputs[step % 6])
        quantize_rows(x, out=(qc, qs))
        dequantize_rows(qc, qs, out=back)
        int8_scores(qc, qs, rc, rs, out=out)
        quantize_rows(x, slots=slots, out=(rc, rs))  # changes rows for the next step
        kept.append((qc.clone(), qs.clone(), back.clone(), out[:, ::97].clone(), rc[slots].clone()))
    rc, rs = _codes(n, d, seed=n)
    cols = torch.arange(0, n, 97, device=DEV)
    for step, (c, s, b, got, written) in enumerate(kept):
        _check_plain(inputs[step % 6], c, s)
        assert torch.equal(b, c.float() * s[:, None])
        _check_scores(got, c, s, rc[cols], rs[cols], None, torch.float32)
        rc[slots], rs[slots] = c, s
        assert torch.equal(written, c)
