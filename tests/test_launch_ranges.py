"""Layer norm and linear over more rows and columns than one launch's work-items count.

A dispatch counts its work-items in 32 bits; longer calls go in several launches.
"""

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp
from tests.test_launch_plan import _run

gpu = pytest.mark.gpu


def test_workgroups_of_a_launch(tmp_path):
    """Below 2^32 work-items for every workgroup, and slices whose pieces begin on whole workgroups."""
    _run(tmp_path, """
  for (int threads = 64; threads <= 1024; threads *= 2) {
    const int64_t most = fh::most_groups(threads);
    CHECK(most * threads < (int64_t{1} << 32) && most >= (int64_t{1} << 21));
    for (int64_t each = 1; each <= 4; each *= 4) {
      const int64_t sizes[] = {most * each, most * each + 1, (int64_t{1} << 31) - 1};
      for (const int64_t rows : sizes) {
        int64_t next = 0;
        const int status = fh::in_slices(rows, most * each, [&](int64_t first, int64_t count) {
          CHECK(first == next && first % each == 0 && (count + each - 1) / each * threads < (int64_t{1} << 32));
          next += count;
          return 0;
        });
        CHECK(status == 0 && next == rows);
      }
    }
  }
""")


def test_rows_of_a_product_launch(tmp_path):
    _run(tmp_path, """
  for (int64_t n = 1; n < (int64_t{1} << 22); n += n < 300 ? 1 : n / 3) {
    const int64_t rows = fh::most_product_rows(n);
    CHECK(rows >= (int64_t{1} << 14) && rows % 128 == 0);
    CHECK(rows / 128 * ((n + 127) / 128) * 512 < (int64_t{1} << 32));
    if (n <= 32) CHECK(rows / 64 * 256 < (int64_t{1} << 32));
  }
""")


def _normal(*shape, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)


@gpu
def test_layer_norm_of_more_rows_than_a_launch():
    """2^26 + 5 rows, 64 work-items each: every row has the bits that it has in a shorter call."""
    rows, cols, part = 2**26 + 5, 2, 2**23
    x, g = _normal(rows, cols, seed=1), _normal(rows, cols, seed=2)
    w, b = _normal(cols, seed=3), _normal(cols, seed=4)
    leaf = x.requires_grad_()
    y = fh.layer_norm(leaf, w, b)
    (dx,) = torch.autograd.grad(y, leaf, g)
    for first in range(0, rows, part):
        piece = x[first : first + part].detach().requires_grad_()
        want = fh.layer_norm(piece, w, b)
        assert torch.equal(y[first : first + part], want)
        (want_dx,) = torch.autograd.grad(want, piece, g[first : first + part])
        assert torch.equal(dx[first : first + part], want_dx)


@gpu
def test_layer_norm_parameters_of_more_columns_than_a_launch():
    """One row of 2^27 + 67 columns: db is g, and dw is g times the normalised row."""
    cols = 2**27 + 67
    x, g = _normal(1, cols, seed=1), _normal(1, cols, seed=2)
    w, b = (torch.full((cols,), v, device="cuda", dtype=torch.bfloat16).requires_grad_() for v in (1.0, 0.0))
    n = fh.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(n, (w, b), g)
    assert torch.equal(db, g[0])
    want = g[0].float() * n[0].detach().float()  # n is rounded to bf16, dw as well
    assert bool(((dw.float() - want).abs() <= 2 * half_ulp(dw.dtype) * want.abs() + floor(dw.dtype)).all())


@gpu
def test_linear_of_more_rows_than_a_launch():
    """2^29 + 70 rows of 8 into 1: every row has the bits that it has in a shorter call."""
    rows, part = 2**29 + 70, 2**26
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-8, 9, (rows, 8), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    w, b, res, g = _normal(1, 8, seed=2), _normal(1, seed=3), _normal(rows, 1, seed=4), _normal(rows, 1, seed=5)
    leaf = x.requires_grad_()
    y = fh.linear(leaf, w, b, activation="silu", residual=res)
    (dx,) = torch.autograd.grad(y, leaf, g)
    y = y.detach()
    for first in range(0, rows, part):
        piece = x[first : first + part].detach().requires_grad_()
        want = fh.linear(piece, w, b, activation="silu", residual=res[first : first + part])
        (want_dx,) = torch.autograd.grad(want, piece, g[first : first + part])
        assert torch.equal(y[first : first + part], want) and torch.equal(dx[first : first + part], want_dx)
