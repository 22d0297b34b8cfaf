"""Clipping in calls that its kernels do not take, or take with care: transforms, tracing, lazy clones, wide types."""

import pytest
import torch

import flash_hypercons as fh

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def _normal(*shape, device="cpu", seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(device, dtype)


# ---- function transforms ---------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
def test_clipping_each_sample_under_vmap(device):
    """vmap over clip_grad_norm and grad_norm is the loop over samples, within FP32's rounding."""
    a, b = _normal(5, 7, 3, device=device), _normal(5, 11, device=device, seed=1)
    clipped, norm = torch.func.vmap(lambda s, t: fh.clip_grad_norm([s, t], 0.5))(a, b)
    alone = torch.func.vmap(lambda s, t: fh.grad_norm([s, t]))(a, b)
    for i in range(5):
        want, want_norm = fh.clip_grad_norm([a[i], b[i]], 0.5)
        torch.testing.assert_close(norm[i], want_norm, rtol=2.0**-22, atol=0)
        torch.testing.assert_close(alone[i], want_norm, rtol=2.0**-22, atol=0)
        for got, w in zip(clipped, want):
            torch.testing.assert_close(got[i], w, rtol=2.0**-21, atol=0)


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_tangents(device):
    """The tangent of the norm along v is <g, v> / norm."""
    g, v = _normal(40, device=device), _normal(40, device=device, seed=1)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(g, v)
        norm, tangent = torch.autograd.forward_ad.unpack_dual(fh.grad_norm([dual]))
    want = (g.double() * v.double()).sum() / g.double().norm()
    assert tangent is not None
    assert abs(tangent.double() - want) <= 2.0**-20 * (g * v).double().abs().sum() / g.double().norm()
