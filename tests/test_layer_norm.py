"""layer_norm against its formula in 64 bits, elementwise.

Bounds: u = 2^-24.  A sum over a row is a chain of at most T = 88 additions a value (a lane's 64
terms, a butterfly of 6, at most 16 wavefronts; longer rows go a vector at a time), so the mean is
off by T u mean|x| and 1 / deviation by (T + 8) u, relative.  With n the normalised value,
err(n) = u (((T + 2) mean|x| + 2 |x|) / deviation + (T + 8) |n|); the rest follows by propagation.
The storage type adds half an ulp of the result, and half a subnormal step.
"""

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp

U, T = 2.0**-24, 88
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def _formula(x, w, b, g, eps):
    """(y, dx, dw, db) and elementwise bounds of each, in 64 bits."""
    x, g = x.double().cpu(), g.double().cpu()
    c = x.shape[-1]
    w = torch.ones(c).double() if w is None else w.double().cpu()
    b = torch.zeros(c).double() if b is None else b.double().cpu()
    d = x - x.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = d * r
    en = U * (((T + 2) * x.abs().mean(-1, keepdim=True) + 2 * x.abs()) * r + (T + 8) * n.abs())
    y = n * w + b
    ey = en * w.abs() + 2 * U * ((n * w).abs() + b.abs())
    q = g * w
    c1, c2 = q.mean(-1, keepdim=True), (q * n).mean(-1, keepdim=True)
    dx = r * (q - c1 - n * c2)
    mq, mqn = q.abs().mean(-1, keepdim=True), (q * n).abs().mean(-1, keepdim=True)
    edx = r * (U * (T * mq + 8 * q.abs() + (T + 8) * n.abs() * mqn) + en * c2.abs()
               + n.abs() * (q.abs() * en).mean(-1, keepdim=True)) + (T + 8) * U * dx.abs()
    flat = lambda v: v.reshape(-1, c)  # noqa: E731
    gn, g2 = flat(g * n), flat(g)
    chain = g2.shape[0] // 256 + 48  # rows a lane adds, row groups, partial rows
    dw, db = gn.sum(0), g2.sum(0)
    edw = chain * U * gn.abs().sum(0) + flat(g.abs() * en).sum(0)
    edb = chain * U * g2.abs().sum(0)
    return (y, dx, dw, db), (ey, edx, edw, edb)


def _check(got, want, bound, what):
    dt = got.dtype
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    limit = half_ulp(dt) * want.abs() + (1 + half_ulp(dt)) * bound + floor(dt)
    off = (got - want).abs()
    assert bool((off <= limit).all()), f"{what}: {(off / limit).max().item():.2f} times the bound"


def _step(x, w, b, g, eps=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = fh.layer_norm(*leaves, eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], g)
    grads = list(grads)
    return y, [grads.pop(0) if t is not None else None for t in leaves]


def _compare(x, w, b, g, eps=1e-5):
    y, grads = _step(x, w, b, g, eps)
    want, bound = _formula(x, w, b, g, eps)
    assert y.is_contiguous() and y.dtype == x.dtype
    _check(y, want[0], bound[0], "y")
    for name, got, i in (("dx", grads[0], 1), ("dw", grads[1], 2), ("db", grads[2], 3)):
        if got is not None:
            _check(got, want[i], bound[i], name)
    with torch.no_grad():
        assert torch.equal(fh.layer_norm(x, w, b, eps), y.detach())


def _inputs(shape, dtype, params=None, seed=0, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device=device)  # noqa: E731
    params, c = params or dtype, shape[-1]
    x = (normal(*shape) * (1 + normal(*shape[:-1], 1).abs()) + 0.5).to(dtype)
    return x, (1 + 0.2 * normal(c)).to(params), (0.3 * normal(c)).to(params), normal(*shape).to(dtype)


# Around the edges of a vector, of each row layout and of the long-row kernels.
COLS = [1, 2, 3, 7, 8, 9, 63, 64, 255, 257, 511, 513, 1023, 1027, 2048, 2052, 4095, 4096, 4104, 8193, 16384, 16385,
        32768, 32771, 40000]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cols", COLS)
def test_widths(cols, dtype):
    _compare(*_inputs((5, cols), dtype, seed=cols))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 255, 256, 257, 4099, 8200])
def test_rows(rows, dtype):
    _compare(*_inputs((rows, 264), dtype, seed=rows))
    if rows < 300:
        _compare(*_inputs((rows, 4096), dtype, seed=rows))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("cols", [40, 1023, 20000])
def test_float32_parameters_beside_16_bit_rows(cols, dtype):
    x, w, b, g = _inputs((9, cols), dtype, torch.float32)
    _compare(x, w, b, g)
    _, (dx, dw, db) = _step(x, w, b, g)
    assert dx.dtype == dtype and dw.dtype == db.dtype == torch.float32


@gpu
@pytest.mark.parametrize("cols", [100, 40000])
def test_missing_parameters(cols):
    x, w, b, g = _inputs((7, cols), torch.float32)
    for ww, bb in ((None, None), (w, None), (None, b)):
        _compare(x, ww, bb, g)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views(dtype):
    t, n, c = 6, 3, 130
    x, w, b, g = _inputs((t, n, c), dtype)
    _compare(x, w, b, g)  # leading dimensions
    _compare(x[:, 1], w, b, g[:, 2])  # one stream of several, in place
    wide, _, _, gw = _inputs((t, c + 5), dtype, seed=1)
    _compare(wide[:, 3:3 + c], w, b, gw[:, 1:1 + c])  # rows at odd elements
    _compare(wide[:, :c].t().contiguous().t(), w, b, g[:, 0])  # columns apart
    _compare(x[:1, 0].expand(t, c), w, b, g[:1, 0].expand(t, c))  # one row for all
    _compare(x[:, 0], w.repeat_interleave(2)[::2], b.flip(0).flip(0), g[:, 0])  # strided parameters
    if dtype == torch.float32:
        neg = torch.complex(g, x).conj().imag
        assert neg.is_neg()
        _compare(neg, w, b, g)


@gpu
def test_neighbours_of_the_rows_are_left_alone():
    x, w, b, g = _inputs((6, 129), torch.bfloat16)
    for fill in (float("inf"), float("nan")):
        pads = [torch.full((6, 140), fill, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        pads[0][:, 5:134], pads[1][:, 3:132] = x, g
        _compare(pads[0][:, 5:134], w, b, pads[1][:, 3:132])


@gpu
def test_rows_far_from_zero_keep_their_variance():
    x, w, b, g = _inputs((4, 1000), torch.float32)
    _compare(x + 4096.0, w, b, g)


@gpu
def test_constant_rows_and_single_columns():
    x = torch.full((3, 77), 2.5, device="cuda")
    w, b, g = torch.ones(77, device="cuda"), torch.full((77,), 0.25, device="cuda"), torch.ones(3, 77, device="cuda")
    y, (dx, dw, _) = _step(x, w, b, g)
    assert torch.equal(y, torch.full_like(y, 0.25)) and not dw.any() and dx.abs().max() < 1e-2
    y, (dx, dw, db) = _step(x[:, :1], w[:1], b[:1], g[:, :1])
    assert torch.equal(y, torch.full_like(y, 0.25)) and not dx.any() and not dw.any() and db.item() == 3.0


@gpu
@pytest.mark.parametrize("cols", [100, 9000])
def test_nan_and_infinity_stay_in_their_row(cols):
    x, w, b, g = _inputs((8, cols), torch.float32)
    x[2, 7], x[5, cols - 1] = float("nan"), float("inf")
    y, (dx, _, db) = _step(x, w, b, g)
    good = torch.tensor([0, 1, 3, 4, 6, 7], device="cuda")
    for t in (y, dx):
        assert t[2].isnan().all() and t[5].isnan().any() and t[good].isfinite().all()
    want, bound = _formula(x[good], w, b, g[good], 1e-5)
    _check(y[good], want[0], bound[0], "y")
    _check(dx[good], want[1], bound[1], "dx")
    assert db.isfinite().all()


@gpu
def test_no_rows():
    x, w, b, g = _inputs((0, 40), torch.float32)
    y, (dx, dw, db) = _step(x, w, b, g)
    assert y.shape == dx.shape == (0, 40) and not dw.any() and not db.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_results_are_the_same_bits_again(dtype):
    args = _inputs((3000, 520), dtype)
    first, again = _step(*args), _step(*args)
    assert torch.equal(first[0], again[0]) and all(map(torch.equal, first[1], again[1]))


@gpu
def test_gradients_against_differences():
    """Central differences of sum(g y) along random directions, h = 2^-6: h^2 / 6 times the third
    derivative (below 20 for these inputs of deviation about 1) and u / h times sum|g y| (about 40
    entries' worth of 2^-18) stay below 2e-2 of the gradient's norm."""
    x, w, b, g = _inputs((4, 48), torch.float32, seed=4)
    _, grads = _step(x, w, b, g)
    for i, (t, d) in enumerate(zip((x, w, b), grads)):
        v = torch.randn(t.shape, device="cuda")
        h = 2.0**-6
        args = [x, w, b]
        value = []
        for sign in (1, -1):
            args[i] = t + sign * h * v
            value.append((fh.layer_norm(*args).double() * g.double()).sum())
        slope = (value[0] - value[1]) / (2 * h)
        want = (d.double() * v.double()).sum()
        assert abs(slope - want) <= 2e-2 * d.double().norm() * v.double().norm() / t.numel()**0.5 + 2e-3 * abs(want)


@gpu
def test_second_derivatives_and_transforms_go_native():
    x, w, b, g = _inputs((3, 20), torch.float32)
    x, w = x.requires_grad_(), w.requires_grad_()

    def grads(norm):
        y = norm(x, w, b)
        dx, dw = torch.autograd.grad(y, (x, w), g, create_graph=True)
        return dx, dw, *torch.autograd.grad(dx.square().sum() + dw.square().sum(), (x, w))

    native = lambda a, ww, bb: torch.nn.functional.layer_norm(a, (20,), ww, bb, 1e-5)  # noqa: E731
    for a, e in zip(grads(fh.layer_norm), grads(native)):
        torch.testing.assert_close(a, e, rtol=1e-4, atol=1e-4)
    per_row = torch.func.vmap(lambda r: fh.layer_norm(r, w, b))(x)
    torch.testing.assert_close(per_row, native(x, w, b), rtol=1e-5, atol=1e-5)


@gpu
def test_compiled_step_matches():
    x, w, b, g = _inputs((33, 72), torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.compile(lambda *a: fh.layer_norm(*a), fullgraph=True, backend="aot_eager")(*leaves)
    got = torch.autograd.grad(y, leaves, g)
    want_y, want = _step(x, w, b, g)
    assert torch.equal(y, want_y) and all(map(torch.equal, got, want))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_cpu_tensors_go_native(dtype):
    x, w, b, g = _inputs((5, 33), dtype, device="cpu")
    _compare(x, w, b, g)


def test_refusals_on_the_cpu():
    with pytest.raises(RuntimeError):
        fh.layer_norm(torch.ones(2, 3), torch.ones(4))


@gpu
def test_refusals():
    x, w, b, _ = _inputs((4, 10), torch.bfloat16)
    with pytest.raises(RuntimeError, match="weight and bias"):
        fh.layer_norm(x, w[:9], b)
    with pytest.raises(RuntimeError, match="weight and bias"):
        fh.layer_norm(x, w, b.half())
    with pytest.raises(RuntimeError, match="one type"):
        fh.layer_norm(x, w, b.float())
    ops = torch.ops.flash_hypercons
    y, stats = ops._layer_norm_forward(x, w, b, 1e-5)
    with pytest.raises(RuntimeError, match="grad must match"):
        ops._layer_norm_backward(y[:3], x, w, b, stats, True, True)
    with pytest.raises(RuntimeError, match="statistics"):
        ops._layer_norm_backward(y, x, w, b, stats[:2], True, True)
