"""Codes of weighted rows against the rational quotient: halves of products of 48 bits, and products that leave the range
of fp32 at its lower end.  code = rint(127 u / max|u|), ties to even, with u = v * w as a rational number: equal."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from circuit_rag.int8 import quantize_rows, rms_norm_quantize

pytestmark = pytest.mark.gpu

DEV = "cuda"
NORM_SCALE_RTOL = 2.5e-6  # as for every norm: four roundings and an fp32 sum of squares


def _rational(v, w):
    """Codes and maximum of one row by fractions."""
    u = [Fraction(float(a)) * Fraction(float(b)) for a, b in zip(v, w)]
    top = max(abs(x) for x in u)
    if top == 0:
        return [0] * len(u), top
    return [round(127 * x / top) for x in u], top  # round() of a fraction takes ties to even


def _check(rows, w, codes, scales, eps):
    rows, w, codes, scales = rows.double().cpu(), w.double().cpu(), codes.cpu().tolist(), scales.cpu().tolist()
    for v, got, scale in zip(rows, codes, scales):
        want, top = _rational(v.tolist(), w.tolist())
        off = [(i, a, b) for i, (a, b) in enumerate(zip(got, want)) if a != b]
        assert not off, off[:8]
        if top == 0:
            assert scale == 0
            continue
        square = sum(Fraction(x) ** 2 for x in v.tolist()) / len(got) + Fraction(eps)
        e = max(square.numerator.bit_length() - square.denominator.bit_length(), -3000) // 2 * 2  # square / 2^e is near one
        exact = float(top / 127 / Fraction(2) ** (e // 2)) / float(square / Fraction(2) ** e) ** 0.5
        assert abs(scale - exact) <= NORM_SCALE_RTOL * exact + 2.0 ** -149


@pytest.mark.parametrize("repeat", [1, 700])
@pytest.mark.parametrize("d", [48, 51, 260, 384, 1000, 5000])
def test_halves_of_weighted_rows(d, repeat):
    rng = np.random.default_rng(d)
    rows, w = np.zeros((4, d), np.float32), np.zeros(d, np.float32)
    w[:] = rng.uniform(0.5, 2, d).astype(np.float32)
    ties = np.arange(d) % 3 != 0
    w[ties] = w[0]
    for r in range(4):
        # maxima 127 k w of up to 48 bits: every (n + 1/2) k w is a half
        k = float(rng.integers(1 << 15, 1 << 16) | 1)
        n = rng.integers(0, 127, d)
        rows[r] = np.where(ties, (2 * n + 1) * k / 2 * rng.choice([-1, 1], d), 60 * k * rng.uniform(-1, 1, d))
        rows[r, 0] = 127 * k
    rows *= (2.0 ** np.array([-20, 0, 9, -60]))[:, None].astype(np.float32)
    x, wt = torch.from_numpy(rows).to(DEV), torch.from_numpy(w).to(DEV)
    codes, scales, _ = rms_norm_quantize(x.repeat(repeat, 1), weight=wt, eps=1e-6)
    _check(x, wt, codes[:4], scales[:4], float(np.float32(1e-6)))
    assert torch.equal(codes, codes[:4].repeat(repeat, 1)) and torch.equal(scales, scales[:4].repeat(repeat))


def test_half_of_the_maximum_of_weighted_rows():
    """u = max / 2, the half that is there for any maximum: 63.5 goes to 64."""
    rng = np.random.default_rng(1)
    v = rng.uniform(1, 2, (2000, 1)).astype(np.float32)
    w = np.array([1.7654321] * 8 + [1.7654321 / 2] * 8, np.float32)
    x = torch.from_numpy(np.concatenate([v, v / 2] * 4 + [v, -v] * 4, 1)).to(DEV)
    codes, _, _ = rms_norm_quantize(x, weight=torch.from_numpy(w).to(DEV))
    assert torch.equal(codes, torch.tensor([127, 64] * 4 + [64, -64] * 4, dtype=torch.int8, device=DEV).expand(2000, 16))


@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("repeat", [1, 500])
@pytest.mark.parametrize("d", [16, 45, 250, 384, 1500, 5000])
def test_products_below_the_range(d, repeat, dtype, wtype):
    """Products that fp32 holds with few bits or not at all, among rows of zeros and of usual size."""
    if dtype == torch.float16:
        sizes, weight = [0.0, 1e-6, 1.0, 1e-4, 3e-7, 100.0], 1e-38  # 16-bit values go down to 6e-8
    else:
        sizes, weight = [0.0, 1e-22, 1.0, 3e-25, 1e-30, 1e-20], 1e-21
    g = torch.Generator().manual_seed(d)
    base = torch.randn(len(sizes), d, generator=g).double() * torch.tensor(sizes).double()[:, None]
    x = base.to(dtype).to(DEV)
    w = (torch.randn(d, generator=g).double() * weight).to(wtype).to(DEV)
    for eps in (0.0, 1e-6):
        codes, scales, _ = rms_norm_quantize(x.repeat(repeat, 1), weight=w, eps=eps)
        _check(x, w, codes[:len(sizes)], scales[:len(sizes)], float(np.float32(eps)))
        assert torch.equal(codes, codes[:len(sizes)].repeat(repeat, 1))
        assert torch.equal(scales, scales[:len(sizes)].repeat(repeat))
    # into slots, with a residual
    slots = torch.tensor([5, -1, 3, 1, 0, 9], device=DEV)
    store = torch.full((6, (d + 15) // 16 * 16), 77, dtype=torch.int8, device=DEV)[:, :d], torch.full((6,), 5.0, device=DEV)
    rms_norm_quantize(x, residual=torch.zeros_like(x), weight=w, eps=0.0, slots=slots, out=store)
    at = [4, 3, 2, 0]  # rows of places 0, 1, 3 and 5
    _check(x[at], w, store[0][[0, 1, 3, 5]], store[1][[0, 1, 3, 5]], 0.0)
    assert (store[0][[2, 4]] == 77).all() and (store[1][[2, 4]] == 5).all()


def test_rows_without_a_weight_keep_their_halves():
    x = (torch.arange(0, 255, device=DEV).float() / 2)[None].repeat(3, 1)
    x[1] *= 1e-40
    x[2] *= 1e30
    x[:, 0] = torch.tensor([127.0, 1e-40 * 127, 1e30 * 127])
    for got in (quantize_rows(x)[0], rms_norm_quantize(x, eps=0.0)[0]):
        for row, codes in zip(x.double().cpu(), got.cpu().tolist()):
            assert codes == _rational(row.tolist(), [1.0] * 255)[0]
