"""relu's gradient where the sums before it are tiny, against the formula in 64 bits.

relu's slope is 1 for every positive sum, however small, and it keeps dz's bits: dz errs only where a
sum's sign may, |z| <= ez, with test_linear's bound ez of a sum's error.  The products and the bias's
sum add test_linear's errors of their own sums.
"""

import pytest
import torch

import flash_hypercons as fh
from tests.test_linear import DTYPES, U, _check, _compare, _inputs, _sum_error

pytestmark = pytest.mark.gpu

# One for each way that sums reach memory: streamed, in tiles, of few terms, in slices, outer products.
SIZES = [(5, 96, 64), (150, 96, 64), (200, 48, 136), (64, 4096, 40), (300, 30, 260)]


def _scaled(m, k, n, dtype, power):
    """Inputs whose sums are about 2^power; FP16 holds neither factor much below 2^-14."""
    x, w, _, _, g = _inputs(m, k, n, dtype, seed=m + n)
    return x * 2.0 ** (power // 2), w * 2.0 ** (power - power // 2), g


def _bounds(x, w, g):
    x, w, g = (t.double().cpu() for t in (x, w, g))
    (rows, k), n = x.shape, w.shape[0]
    return x, w, g, x @ w.t(), rows, k, n


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_relu_gradients_of_tiny_sums(m, k, n, dtype):
    power = -30 if dtype == torch.float16 else -70
    x, w, g = _scaled(m, k, n, dtype, power)
    leaves = [x.requires_grad_(), w.requires_grad_(), torch.zeros(n, device="cuda", dtype=dtype).requires_grad_()]
    y = fh.linear(*leaves, activation="relu")
    dx, dw, db = torch.autograd.grad(y, leaves, g)
    x, w, g, z, rows, k, n = _bounds(x.detach(), w.detach(), g)
    ez = _sum_error(k, dtype) * (x.abs() @ w.abs().t())
    dz = g * (z > 0)
    edz = torch.where(z.abs() <= ez, g.abs(), torch.zeros_like(g))
    size = dz.abs() + edz
    _check(dx, dz @ w, edz @ w.abs() + _sum_error(n, dtype) * (size @ w.abs()), "dx")
    _check(dw, dz.t() @ x, edz.t() @ x.abs() + _sum_error(rows, dtype) * (size.t() @ x.abs()), "dw")
    _check(db, dz.sum(0), edz.sum(0) + (rows + 8) * U * size.sum(0), "db")
    assert bool(db.any())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_zero_sums_have_no_slope(dtype):
    """relu's slope at 0 and at -0 is 0."""
    x = torch.tensor([[0.0, 0.0], [-0.0, 0.0], [2.0**-12, 2.0**-12]], device="cuda", dtype=dtype).requires_grad_()
    w = torch.tensor([[1.0, -1.0]], device="cuda", dtype=dtype)
    y = fh.linear(x, w, activation="relu")
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert not dx.any()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_smooth_activations_of_tiny_sums(act, dtype):
    """Their slope is 1/2 there: within test_linear's bounds."""
    x, w, g = _scaled(150, 96, 64, dtype, -30)
    _compare(x, w, None, None, act, g)
