"""Fp8Matrix.quantize on the GPU: codes and scales at every size of weights, against
the oracle's rounding. No tolerance: dividing by a power of two is exact."""

import pytest
import torch

import trntensor_amd as tt
from oracle import fp8 as ref

pytestmark = pytest.mark.gpu


def _values(mat):
    """The weights that a matrix stands for: its products with the unit vectors, exact in 32 bits."""
    return tt.fp8_matmul(torch.eye(mat.shape[1], dtype=torch.float32).cuda(), mat, dtype=torch.float32).t().cpu().double()


def _want(w):
    """The oracle's values of weights of one block of 128 x 128."""
    e = float(ref.exponent(w.double().abs().max().item()))
    return ref.round_e4m3(w.double() * 2.0 ** -e) * 2.0 ** e


def _halfway(power):
    """Every code's value and the middles between neighbours, of either sign, times
    2^power, in a block whose largest value is 448 2^power."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mids = (codes[1:] + codes[:-1]) / 2
    w = torch.zeros((4, 127), dtype=torch.float64)
    w[0], w[1] = codes, -codes
    w[2, :126], w[3, :126] = mids, -mids
    w[2:, 126] = 448.0
    return w * 2.0 ** power


@pytest.mark.parametrize("first", range(-110, 105, 16))
def test_halfway_weights_go_to_the_even_code(hip, first):
    """Products with the unit vectors need a scale that is a float32: 2^-126 to 2^127."""
    for power in range(first, min(first + 16, 105)):
        w = _halfway(power).float()
        assert torch.equal(w.double(), _halfway(power))
        assert torch.equal(_values(tt.Fp8Matrix.quantize(w.cuda())), _want(w)), power


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("default", [torch.float16, torch.bfloat16, torch.float64])
def test_weights_do_not_depend_on_the_default_dtype(hip, dtype, default):
    g = torch.Generator().manual_seed(5)
    w = (0.0005 * torch.randn((100, 120), generator=g, dtype=torch.float32)).to(dtype)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        mat = tt.Fp8Matrix.quantize(w.cuda())
    finally:
        torch.set_default_dtype(before)
    assert torch.equal(_values(mat), _want(w))
