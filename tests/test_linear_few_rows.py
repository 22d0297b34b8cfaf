"""linear with at most 32 rows or outputs in FP32, against its formula in 64 bits.

The bounds are test_linear's: an FP32 sum of K products of bf16 parts is off by at most
(2 K + 16) u sum|x w|, u = 2^-24.
"""

import pytest
import torch

import flash_hypercons as fh
from tests.test_linear import _check, _compare, _formula, _inputs

pytestmark = pytest.mark.gpu

# Rows or outputs at and around 1, 4 and 32; sums that end inside a strip of 32, a wavefront's
# turn of 128 and a slice; strips of 64 that end inside; widths that are no whole vectors.
SIZES = [
    (1, 4, 4), (1, 32, 64), (1, 36, 68), (1, 1024, 260), (2, 28, 132), (4, 128, 4), (5, 132, 1000),
    (31, 100, 68), (32, 64, 64), (32, 4096, 96), (33, 256, 64), (28, 2052, 516),
    (64, 68, 1), (100, 200, 4), (260, 1000, 32), (1000, 4, 32), (4096, 36, 8), (2052, 300, 33),
    (3, 37, 50), (7, 36, 51), (40, 1027, 5),
]  # fmt: skip


@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(m, k, n):
    x, w, b, res, g = _inputs(m, k, n, torch.float32, seed=m + k + n)
    _compare(x, w, b, res, "silu", g)
    _compare(x, w, None, None, None, g)


@pytest.mark.parametrize("m,n", [(6, 200), (200, 8)])
@pytest.mark.parametrize("pad,offset", [(4, 0), (8, 4), (5, 0), (4, 1), (4, 2)])
def test_rows_apart_and_shifted(pad, offset, m, n):
    """Rows a whole number of vectors apart or not, beginning on one or not; what lies between is NaN."""
    x, w, b, res, g = _inputs(m, 64, n, torch.float32)

    def apart(t):
        wide = torch.full((t.shape[0], t.shape[1] + pad + offset), float("nan"), device="cuda")
        wide[:, offset : offset + t.shape[1]] = t
        return wide[:, offset : offset + t.shape[1]]

    _compare(apart(x), apart(w), b, res, "gelu", g)
    y = fh.linear(apart(x), apart(w))
    want, bound = _formula(x, w, None, None, None, g)
    _check(y, want[0], bound[0], "y")


@pytest.mark.parametrize("m,n", [(4, 128), (128, 4)])
@pytest.mark.parametrize("at", [0, 31, 32, 63, 99])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_not_finite(value, at, m, n):
    x, w, *_ = _inputs(m, 100, n, torch.float32)
    w = w.abs() + 0.5
    x[2, at] = value
    y = fh.linear(x, w)
    clean = x.clone()
    clean[2, at] = 0
    other = [i for i in range(m) if i != 2]
    assert torch.equal(y[other], fh.linear(clean, w)[other])
    assert bool((torch.isnan(y[2]) if value != value else y[2] == value).all())


@pytest.mark.parametrize("m,n", [(4, 128), (128, 4)])
def test_infinity_against_zero_is_nan(m, n):
    x, w, *_ = _inputs(m, 64, n, torch.float32)
    w = w.abs() + 0.5
    x[1, 5] = float("inf")
    w[3, 5] = 0
    y = fh.linear(x, w)
    assert torch.isnan(y[1, 3]) and int(torch.isnan(y).sum()) == 1


@pytest.mark.parametrize("m,k,n", [(2, 4096, 128), (300, 4096, 8)])
def test_the_same_bits_again(m, k, n):
    x, w, b, res, g = _inputs(m, k, n, torch.float32)
    first = [fh.linear(x, w, b, activation="gelu", residual=res) for _ in range(4)]
    assert all(torch.equal(first[0], t) for t in first[1:])


def test_large_and_small_values():
    """Products across 80 powers of two, where terms that a part loses would show."""
    x, w, *_ = _inputs(3, 512, 96, torch.float32)
    scale = 2.0 ** torch.linspace(-40, 40, 512, device="cuda").round()
    x, w = x * scale, w / scale
    g = torch.ones(3, 96, device="cuda")
    want, bound = _formula(x, w, None, None, None, g)
    _check(fh.linear(x, w), want[0], bound[0], "y")


FEW_TERMS = [(130, 1, 200), (256, 31, 132), (300, 32, 129), (129, 33, 260), (500, 5, 70), (70, 32, 1000)]


@pytest.mark.parametrize("m,k,n", FEW_TERMS)
def test_sums_of_few_terms(m, k, n):
    """One step of the sum and just more, tiles that end inside, results at every alignment."""
    x, w, b, res, g = _inputs(m, k, n, torch.float32, seed=m)
    _compare(x, w, b, res, "gelu_tanh", g)
    x, w, b, res, g = _inputs(k, m, n, torch.float32, seed=n)
    _compare(x, w, b, res, None, g)
