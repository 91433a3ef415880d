"""How near linear comes to its definition where element-wise bounds on sums say little."""
import math

import pytest
import torch

from _layers import FLOAT32_SIZES, TINY, U, act, float32_norm_bound, norm_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,n", [(1, 40), (2, 41), (7, 41), (20, 40), (100, 264), (300, 264), (300, 265)])
def test_gelu_of_negative_arguments(cuda, dtype, m, n):
    """gelu is small there, and small against what 1 + erf loses.  The 16-bit form of the normal distribution is the tail
    of formula 7.1.26 (Abramowitz and Stegun), of which the formula's own deviation is allowed, taken here in float64, and
    2^-16 of the value: the exponent, up to 22, is off by 2^-23 of itself; a polynomial whose terms add up to at most 5 times
    its value, with 8 roundings of 2^-24; the hardware's exponential and reciprocal, 2^-21 each."""
    from aimet_b200.v2.nn import linear
    z = (-5.5 + 5.0 * torch.arange(n, device=cuda) / n).to(dtype)
    x = torch.zeros(m, 64, device=cuda, dtype=dtype)
    w = torch.zeros(n, 64, device=cuda, dtype=dtype)
    x[:, 3] = 1
    w[:, 3] = z
    y = linear(x, w, None, "gelu").double()
    z = z.double()
    want = act(z, "gelu")
    t = 1 / (1 + 0.3275911 * z.abs() / math.sqrt(2))
    poly = t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (-1.453152027 + t * 1.061405429))))
    formula = (0.5 * z * poly * torch.exp(-z * z / 2) - want).abs()
    err = (y - want).abs() - (U[dtype] + 2.0 ** -16) * want.abs() - (1 + U[dtype]) * formula - TINY[dtype] / 2
    assert float(err.max()) <= 0, float((y - want).abs().div(want.abs()).max())


@pytest.mark.parametrize("m,k,n", FLOAT32_SIZES)
def test_float32_products_keep_their_operands(cuda, m, k, n):
    """The three products of a float32 layer by their norms: operands of fewer bits would show at every depth."""
    from aimet_b200.v2.nn import linear
    g = torch.Generator(device="cuda").manual_seed(107)
    x, w, dy = (torch.randn(s, device=cuda, generator=g).requires_grad_(True) for s in ((m, k), (n, k), (m, n)))
    y = linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy.detach())
    x, w, dy = x.detach().double(), w.detach().double(), dy.detach().double()
    assert norm_error(y, x @ w.t()) <= float32_norm_bound(k)
    assert norm_error(dx, dy @ w) <= float32_norm_bound(n)
    assert norm_error(dw, dy.t() @ x) <= float32_norm_bound(m)
