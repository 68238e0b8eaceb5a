"""The 8-bit chain from its definitions, in float64 on the CPU (test
infrastructure only): rows in 8 bits, the root-mean-square norm, products of
such rows with 8-bit weights and the gated block on two of them. Nothing is
shared with the product or its plain forms.
"""

from __future__ import annotations

import torch

from .serving import round_e4m3


def exponent(amax: float) -> int:
    """The smallest e >= -127 with amax <= 448 * 2^e."""
    e = -127
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def exponents(x: torch.Tensor) -> torch.Tensor:
    """(rows, blocks) exponents of rows x, from their blocks' largest finite magnitudes."""
    x = torch.where(x.isfinite(), x.double().abs(), 0.0)
    top = torch.stack([x[:, i: i + 128].amax(dim=1) for i in range(0, x.shape[1], 128)], dim=1)
    limits = 448.0 * torch.exp2(torch.arange(-127, 130, dtype=torch.float64))  # exact
    return torch.searchsorted(limits, top.contiguous()) - 127


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes' values and exponents of rows x; infinities become NaN."""
    e = exponents(x)
    y = torch.where(x.isfinite(), x.double(), torch.nan) / spread(torch.exp2(e.double()), x.shape[1])
    return round_e4m3(y), e


def spread(scales: torch.Tensor, columns: int) -> torch.Tensor:
    """(rows, blocks) scales as (rows, columns)."""
    return scales.double()[:, torch.arange(columns) // 128]


def weights(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """(n, k) float64 weights: scales[n // 128, k // 128] * code."""
    n, k = codes.shape
    return codes.double() * scales.double()[torch.arange(n) // 128][:, torch.arange(k) // 128]


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None, eps: float):
    """(norm, h): h = x + residual, over the root of its mean square plus eps."""
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    return (y if weight is None else y * weight.double()), h


def act(a: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "silu":
        return a / (1.0 + torch.exp(-a))
    return 0.5 * a * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3)))
