"""What embedding and the loss compose natively on the GPU: indices out of range give NaN there as in the kernels."""

import pytest
import torch

import flash_hypercons as fh

pytestmark = pytest.mark.gpu
BAD = [3, 100, 499, 7]


def _tokens(vocab, dtype=torch.int64):
    t = torch.randint(0, vocab, (500,), device="cuda")
    t[3], t[100], t[499], t[7] = -1, vocab, 2**31 - 1, -(2**31)
    good = torch.ones(500, dtype=torch.bool, device="cuda")
    good[BAD] = False
    return t.to(dtype), good


@pytest.mark.parametrize("indices", [torch.int64, torch.int32], ids=str)
@pytest.mark.parametrize("streams", [None, 3])
def test_embedding(streams, indices):
    t, good = _tokens(30, indices)
    w = torch.randn(30, 8, dtype=torch.float64, device="cuda", requires_grad=True)
    y = fh.embedding(t, w, scale=2.0, streams=streams, padding_idx=4)
    g = torch.randn_like(y)
    (dw,) = torch.autograd.grad(y, w, g)
    want = fh.embedding(t[good], w, scale=2.0, streams=streams, padding_idx=4)
    assert y[~good].isnan().all() and torch.equal(y[good], want)
    torch.testing.assert_close(dw, torch.autograd.grad(want, w, g[good])[0])


@pytest.mark.parametrize("indices", [torch.int64, torch.int32], ids=str)
@pytest.mark.parametrize("ignore", [-100, 0, 5])
def test_loss(ignore, indices):
    vocab = 20
    t, good = _tokens(vocab, indices)
    t[200:260] = ignore
    x = torch.randn(500, 8, dtype=torch.float64, device="cuda")
    x[t == ignore] = float("nan")
    leaves = [a.requires_grad_() for a in (x, torch.randn(vocab, 8, dtype=torch.float64, device="cuda"),
                                           torch.randn(vocab, dtype=torch.float64, device="cuda"))]
    loss = lambda at, **args: fh.linear_cross_entropy(leaves[0][at], leaves[1], t[at], leaves[2], ignore_index=ignore, **args)  # noqa: E731
    everything = slice(None)
    each = loss(everything, reduction="none")
    dx, dw, db = torch.autograd.grad(each.sum(), leaves)
    want = loss(good, reduction="none")
    assert each[~good].isnan().all() and torch.equal(each[good], want)
    (other,) = torch.autograd.grad(want.sum(), leaves[:1])
    assert dx[~good].isnan().all() and not dx[t == ignore].any() and dw.isnan().all() and db.isnan().all()
    torch.testing.assert_close(dx[good], other[good])
    for reduction in ("sum", "mean"):
        assert loss(everything, reduction=reduction).isnan()
        # As torch's own where every index is in range.
        rows = torch.where((t[good] == ignore)[:, None], 0.0, leaves[0][good])
        native = torch.nn.functional.cross_entropy(torch.nn.functional.linear(rows, leaves[1], leaves[2]), t[good].long(),
                                                   ignore_index=ignore, reduction=reduction)
        got = loss(good, reduction=reduction)
        torch.testing.assert_close(got, native)
        for a, e in zip(torch.autograd.grad(got, leaves), torch.autograd.grad(native, leaves)):
            torch.testing.assert_close(a, e)


def test_no_target():
    x = torch.full((4, 8), float("nan"), dtype=torch.float64, device="cuda", requires_grad=True)
    w = torch.randn(5, 8, dtype=torch.float64, device="cuda", requires_grad=True)
    t = torch.full((4,), -100, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss = fh.linear_cross_entropy(x, w, t, reduction=reduction)
        assert loss.isnan() if reduction == "mean" else not loss.any()
        assert not any(d.any() for d in torch.autograd.grad(loss.sum(), (x, w)))


def test_function_transforms():
    t, good = _tokens(30)
    w = torch.randn(30, 8, device="cuda")
    x = torch.randn(500, 8, device="cuda")
    y = torch.func.vmap(lambda a: fh.embedding(a, w))(t)
    assert y[~good].isnan().all() and torch.equal(y[good], w[t[good]])
    dx = torch.func.grad(lambda a: fh.linear_cross_entropy(a, w, t, reduction="sum"))(x)
    assert dx[~good].isnan().all() and dx[good].isfinite().all()


def test_a_table_without_rows_is_refused():
    t, w = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.empty(0, 8, device="cuda")
    with pytest.raises(IndexError, match="no rows"):
        fh.embedding(t, w)
    with pytest.raises(IndexError, match="no rows"):
        fh.linear_cross_entropy(torch.randn(3, 8, device="cuda"), w, t)
    assert fh.embedding(t[:0], w).shape == (0, 8)
