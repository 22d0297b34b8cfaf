"""gelu of 16-bit results, between -13 and 13, against its definition in 64 bits.

The kernels take Phi(-|z|) from a formula whose relative error grows to the bounds of TAIL
(computed here from the formula itself).  FP32 arithmetic adds (z^2 / 2 + 16) 2^-23 of the result:
the exponent's rounding, and a few operations'.  The storage type adds half an ulp, and half a
subnormal step.
"""

import math

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp

# (z at least, relative error of the formula for Phi(z) at most)
TAIL = [(-1, 3.1e-7), (-2, 3.1e-6), (-3, 5.2e-5), (-4, 4.7e-4), (-5, 1.6e-3), (-6, 3.6e-3), (-8, 1.1e-2), (-13, 3.8e-2)]


def _phi(z):
    """Phi(z) in 64 bits."""
    return 0.5 * torch.special.erfc(-z * math.sqrt(0.5))


def _bound(z):
    bound = torch.full_like(z, TAIL[-1][1])
    for least, relative in reversed(TAIL):
        bound = torch.where(z >= least, relative, bound)
    return bound


def test_formula():
    """Abramowitz and Stegun 7.1.26 in 64 bits keeps to TAIL, and to 7e-8."""
    z = -torch.linspace(0, 13, 130001, dtype=torch.float64)
    t = 1 / (1 - 0.3275911 * math.sqrt(0.5) * z)
    s = (((1.061405429 * t - 1.453152027) * t + 1.421413741) * t - 0.284496736) * t + 0.254829592
    off = (0.5 * s * t * torch.exp(-z * z / 2) - _phi(z)).abs()
    assert bool((off <= _bound(z) * _phi(z)).all()) and off.max() < 7e-8


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_tail(dtype, rows):
    z = torch.linspace(-13, 13, 4096, device="cuda").to(dtype)
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    y = fh.linear(z[:, None], one, activation="gelu") if rows else fh.linear(one, z[:, None], activation="gelu")
    z = z.double().cpu()
    want = z * _phi(z)
    # Beyond 0 the formula's error is that of 1 - Phi(z).
    off = torch.where(z < 0, _bound(z) * want.abs(), _bound(-z) * z * _phi(-z)) + (z * z / 2 + 16) * 2.0**-23 * want.abs()
    limit = (1 + half_ulp(dtype)) * off + half_ulp(dtype) * want.abs() + floor(dtype)
    assert bool(((y.reshape(-1).double().cpu() - want).abs() <= limit).all())
