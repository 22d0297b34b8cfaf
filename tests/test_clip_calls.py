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


# ---- tracing ---------------------------------------------------------------------------


LAYOUTS = {
    "rows": lambda t: t,
    "columns": lambda t: t.t(),
    "permuted": lambda t: t.view(3, 4, 90).permute(2, 0, 1),
    "gapped": lambda t: t[:, 1:40],
    "gapped columns": lambda t: t[:, 1:40].t(),
    "every second": lambda t: t[:, ::2],
    "expanded": lambda t: t[:1].expand(5, 90),
    "one row": lambda t: t[:1, :40],
    "one column": lambda t: t[:, :1],
    "empty": lambda t: t[:0, :4].t(),
    "scalar": lambda t: t[0, 0],
    "negated": lambda t: torch.complex(t, t).conj().imag,
}


@gpu
@pytest.mark.parametrize("layout", LAYOUTS)
def test_traced_results_have_the_real_strides(layout):
    t = LAYOUTS[layout](torch.zeros(12, 90, device="cuda"))
    with torch.no_grad():
        real, _ = fh.clip_grad_norm([t], 1.0)
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        fake, norm = torch.ops.flash_hypercons._clip_grads([mode.from_tensor(t)], 1.0, 2.0)
    assert fake[0].shape == real[0].shape and fake[0].stride() == real[0].stride() and norm.shape == ()


@gpu
def test_compiled_clipping_matches():
    wide, flat = _normal(12, 90, device="cuda"), _normal(33, device="cuda", seed=1, dtype=torch.bfloat16)
    grads = [wide[:, 1:40].t(), wide[:, 50:].t(), flat]

    def clip(*g):
        clipped, norm = fh.clip_grad_norm(g, 0.5)
        return [c.view(-1) if c.is_contiguous() else c.t() for c in clipped], norm

    got, norm = torch.compile(clip, fullgraph=True, backend="aot_eager")(*grads)
    want, want_norm = clip(*grads)
    assert torch.equal(norm, want_norm) and all(map(torch.equal, got, want))


# ---- copy-on-write ---------------------------------------------------------------------


@gpu
def test_lazy_clones_keep_their_own_values():
    kept = _normal(300, device="cuda")
    before = kept.clone()
    params = [torch.nn.Parameter(torch.zeros_like(kept)) for _ in range(2)]
    for p in params:
        p.grad = torch._lazy_clone(kept)
    want, want_norm = fh.clip_grad_norm([before, before], 0.5)
    norm = fh.clip_grad_norm_(params, 0.5)
    assert torch.equal(kept, before)
    assert torch.equal(norm, want_norm) and all(torch.equal(p.grad, w) for p, w in zip(params, want))


# ---- wide types, which go native -------------------------------------------------------


@pytest.mark.parametrize("scale", [1.0, 1e60, 1e-60])
@pytest.mark.parametrize("device", DEVICES)
def test_float64_gradients_are_scaled_in_float64(device, scale):
    """The norm and the factor are a few FP64 roundings off, 2^-53 each, and sums of 58 squares."""
    grads = [_normal(40, device=device, dtype=torch.float64) * scale,
             _normal(2, 9, device=device, seed=1, dtype=torch.float64) * scale]
    norm = torch.cat([g.reshape(-1) for g in grads]).norm()
    limit = 0.25 * float(norm)
    factor = limit / (norm + 1e-6) if scale >= 1.0 else torch.ones_like(norm)
    clipped, got = fh.clip_grad_norm(grads, limit if scale >= 1.0 else 1.0)
    assert got.dtype == torch.float32 and torch.equal(got, norm.float())
    for c, g in zip(clipped, grads):
        assert c.dtype == torch.float64
        torch.testing.assert_close(c, g * factor, rtol=2.0**-45, atol=0)


@pytest.mark.parametrize("p", [1.0, 2.0, 3.0, float("inf")])
@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128], ids=str)
def test_complex_gradients_are_scaled_whole(dtype, p):
    real, imag = _normal(40), _normal(40, seed=1)
    g = torch.complex(real, imag).to(dtype)
    norm = torch.linalg.vector_norm(g.to(torch.complex128), p)
    clipped, got = fh.clip_grad_norm([g], 0.25 * float(norm), p)
    torch.testing.assert_close(got.double(), norm, rtol=2.0**-22, atol=0)
    torch.testing.assert_close(clipped[0], (g.to(torch.complex128) * 0.25).to(dtype), rtol=1e-5, atol=0)
    param = torch.nn.Parameter(torch.zeros_like(g))
    param.grad = g.clone()
    fh.clip_grad_norm_([param], 0.25 * float(norm), p)
    assert torch.equal(param.grad, clipped[0])
