"""The root-mean-square norm of rows whose squares 32 bits do not hold: large ones whose
sum passes 2^128 (up to the documented 2^63 an element), and small ones with an eps as small
or none, whose squares fall below 2^-126.

Tolerances, fixed before the first run: those of the norm elsewhere, (K / 512 + 20) 2^-24 and
the result's rounding, for products with a power of two are exact: the factor that brings
the larger of a row's top and eps's root to 1 loses nothing but what is 2^-126 of it, whose
square is nothing next to the sum. Results below 2^-126 are off by 2^-149."""

import math

import pytest
import torch

import trntensor_amd as tt
from oracle import fp8 as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# A wavefront a row, a workgroup a row with one, two, four and eight passes, and rows read again.
WIDTHS = [1, 40, 511, 1000, 2048, 2300, 8192, 16384, 20000]


def _rows(m, k, power, dtype, seed):
    """Magnitudes of 2^(power - 1) to 0.99 2^power, of either sign."""
    g = torch.Generator().manual_seed(seed)
    x = (0.5 + 0.49 * torch.rand((m, k), generator=g)) * (torch.randint(0, 2, (m, k), generator=g) * 2 - 1)
    return torch.ldexp(x, torch.tensor(power)).to(dtype)


def _check(x, weight, residual, eps, fp8):
    dev = [None if t is None else t.cuda() for t in (x, weight, residual)]
    got = tt.rms_norm(dev[0], dev[1], residual=dev[2], eps=eps, fp8=fp8)
    got, total = got if residual is not None else (got, None)
    k = x.shape[-1]
    want, h = ref.rms_norm(x, weight, residual, eps)
    rel = (k / 512 + 20) * 2.0 ** -24
    if total is not None:
        assert ((total.cpu().double() - h).abs() <= U[x.dtype] * 1.01 * h.abs() + 2.0 ** -134).all()
    if not fp8:
        tol = (rel + U[x.dtype]) * 1.01 * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -134)
        assert ((got.cpu().double() - want).abs() <= tol).all()
        return
    scales = ref.spread(got.scales.float().cpu(), k)
    value = got.codes.float().cpu().double() * scales
    assert ((value - want).abs() <= 2.0 ** -4 * 1.01 * want.abs() + 2.0 ** -10 * scales).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", WIDTHS)
def test_large_rows(hip, k, dtype, fp8):
    weight = 1.0 + 0.1 * torch.rand(k, generator=torch.Generator().manual_seed(k))
    for power in (50, 57, 58, 60, 62, 63):
        x = _rows(3, k, power, dtype, k + power)
        _check(x, weight, None, 1e-6, fp8)
        x[1] = 0.0  # one large element in a small row, and a row of zeros beside them
        x[2] = 1.0
        x[2, k // 2] = 2.0 ** (power - 1)
        _check(x, None, None, 1e-6, fp8)
        half = _rows(3, k, power - 2, dtype, k + power)
        _check(half, weight, half.flip(0), 1e-6, fp8)
    _check(_rows(2, k, 60, dtype, k), weight, None, 1e37, fp8)  # where eps counts


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", WIDTHS)
def test_small_rows(hip, k, dtype, fp8):
    """eps none, below the row's mean square, next to it and above it."""
    weight = 1.0 + 0.1 * torch.rand(k, generator=torch.Generator().manual_seed(k))
    for power in (-45, -52, -60, -66, -75, -90, -110, -125):
        x = _rows(3, k, power, dtype, k - power)
        for eps in (0.0, 4.0 ** (power - 4), 4.0 ** power, 4.0 ** (power + 5)):
            _check(x, weight, None, eps, fp8)
        _check(x, None, x.flip(0).roll(1, 1) * 0.5, 4.0 ** power, fp8)
    x = _rows(2, k, -140, torch.float32, k)  # below the type's smallest normal
    _check(x, weight, None, 0.0, fp8)
    _check(x, weight, None, 1e-31, False)


def test_small_rows_float16(hip):
    for k in (40, 2048):
        x = _rows(3, k, -20, torch.float16, k)
        for eps in (0.0, 1e-13, 1e-50):
            _check(x, None, None, eps, False)


@pytest.mark.parametrize("k", WIDTHS)
def test_rows_of_zeros_and_beyond(hip, k):
    x = torch.zeros((2, k)).cuda()
    for eps in (1e-6, 1e-30, 1e-44, 1e-50, 1e-200, 5e-324):
        assert not tt.rms_norm(x, eps=eps).any()
        rows = tt.rms_norm(x, eps=eps, fp8=True)
        assert not rows.codes.float().any()
    assert tt.rms_norm(x, eps=0.0).isnan().all()  # 0 / 0
    for value in (math.inf, -math.inf, math.nan):  # as ever, next to large and small values
        for other in (2.0 ** 60, 2.0 ** -70):
            y = torch.full((1, k), other)
            y[0, k // 3] = value
            z = tt.rms_norm(y.cuda(), eps=0.0).cpu()
            assert z[0, k // 3].isnan()
            rest = torch.arange(k) != k // 3
            assert z[0, rest].isnan().all() if math.isnan(value) else not z[0, rest].any()
