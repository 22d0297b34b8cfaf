"""linear against its formula in 64 bits, elementwise.

Bounds: u = 2^-24.  A sum of K products is off by at most (K + 8) u sum|x w| (any order, FP32
accumulators); FP32 operands, multiplied as sums of bf16 parts with the products below 2^-22 left
out, by (2 K + 16) u sum|x w|.  The activations' slopes stay below 1.13 and their curvatures below
1.2; computing them costs 8 u.  The backward's z is FP16 for 16-bit types (2^-11), and dz is rounded
to the storage type.  The storage type adds half an ulp of the result, and half a subnormal step.
"""

import math

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp

U = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
gpu = pytest.mark.gpu


def _act(z, act):
    """(act(z), act'(z)) in 64 bits."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z**3))
        return z * (1 + t) / 2, (1 + t) / 2 + z / 2 * (1 - t * t) * k * (1 + 0.134145 * z * z)
    if act == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    return z, torch.ones_like(z)


def _sum_error(k, dtype):
    return ((2 * k + 16) if dtype == torch.float32 else (k + 8)) * U


def _formula(x, w, b, res, act, g):
    """Results and elementwise bounds in 64 bits: y, dx, dw, db."""
    dtype = x.dtype
    k, rows = x.shape[-1], x[..., 0].numel()
    x, w = x.double().cpu().reshape(-1, k), w.double().cpu()
    n = w.shape[0]
    z = x @ w.t()
    ez = _sum_error(k, dtype) * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b.double().cpu()
        ez = ez + 2 * U * z.abs()
    y, slope = _act(z, act)
    ey = 1.13 * ez + (8 * U * z.abs() if act else 0)
    if res is not None:
        y = y + res.double().cpu().reshape(-1, n)
        ey = ey + 2 * U * y.abs()
    g = g.double().cpu().reshape(-1, n)
    dz = g * slope
    edz = torch.zeros_like(dz)
    if act:
        step = 0.0 if dtype == torch.float32 else 2.0**-11
        edz = g.abs() * (1.2 * (ez + step * z.abs() + 2.0**-25) + 16 * U)
        if act == "relu":  # a step: it errs only where the sum's sign may
            edz = torch.where(z.abs() <= ez + 2.0**-25, g.abs(), torch.zeros_like(z))
    rounded = edz + (half_ulp(dtype) * (dz.abs() + edz) + floor(dtype) if act else 0)
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    size = dz.abs() + rounded
    edx = rounded @ w.abs() + _sum_error(n, dtype) * (size @ w.abs())
    edw = rounded.t() @ x.abs() + _sum_error(rows, dtype) * (size.t() @ x.abs())
    edb = edz.sum(0) + (rows + 8) * U * (dz.abs() + edz).sum(0)
    return (y, dx, dw, db), (ey, edx, edw, edb)


def _check(got, want, bound, what):
    dt = got.dtype
    got = got.detach().double().cpu().reshape(want.shape)
    limit = half_ulp(dt) * want.abs() + (1 + half_ulp(dt)) * bound + floor(dt)
    off = (got - want).abs()
    assert bool((off <= limit).all()), f"{what}: {(off / limit).max().item():.2f} times the bound"


def _step(x, w, b, res, act, g):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, res)]
    y = fh.linear(*leaves[:3], activation=act, residual=leaves[3])
    grads = list(torch.autograd.grad(y, [t for t in leaves if t is not None], g))
    return y, [grads.pop(0) if t is not None else None for t in leaves]


def _compare(x, w, b, res, act, g):
    y, (dx, dw, db, dres) = _step(x, w, b, res, act, g)
    want, bound = _formula(x, w, b, res, act, g)
    assert y.is_contiguous() and y.dtype == x.dtype and y.shape == (*x.shape[:-1], w.shape[0])
    for name, got, i in (("y", y, 0), ("dx", dx, 1), ("dw", dw, 2), ("db", db, 3)):
        if got is not None:
            _check(got, want[i], bound[i], name)
    assert dres is None or torch.equal(dres, g)
    with torch.no_grad():
        assert torch.equal(fh.linear(x, w, b, activation=act, residual=res), y.detach())


def _inputs(m, k, n, dtype, seed=0, device="cuda", bias=None):
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device=device)  # noqa: E731
    x, w = normal(m, k).to(dtype), (normal(n, k) * k**-0.5).to(dtype)
    return x, w, normal(n).to(bias or dtype), normal(m, n).to(dtype), normal(m, n).to(dtype)


# Around the edges of vectors, tiles and slices, from one of each to several tiles.
SIZES = [(1, 1, 1), (1, 8, 8), (3, 7, 5), (1, 64, 129), (2, 4096, 64), (16, 200, 48), (17, 136, 24), (64, 1000, 16),
         (127, 65, 130), (128, 128, 128), (129, 264, 257), (250, 72, 1030), (300, 2056, 8), (513, 520, 264),
         (1000, 16, 2000), (33, 8200, 40), (1025, 96, 9), (256, 512, 512), (300, 768, 640), (520, 1111, 777)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(m, k, n, dtype):
    x, w, b, res, g = _inputs(m, k, n, dtype, seed=m + k + n)
    act = ACTS[(m + k + n) % 5]
    _compare(x, w, b, res if (m + n) % 2 else None, act, g)


# Enough tiles of 256 for y, dx or dW, with ragged edges in every dimension.
LARGE = [(4000, 203, 3990), (3990, 4001, 263), (264, 4000, 3990)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", LARGE)
def test_large_sizes(m, k, n, dtype):
    _compare(*_inputs(m, k, n, dtype, seed=m + k)[:4], "gelu" if k == 203 else None, _inputs(m, k, n, dtype)[4])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 40, 260])
def test_activations(m, act, dtype):
    x, w, b, res, g = _inputs(m, 144, 136, dtype, seed=m)
    _compare(3 * x, w, b, res, act, g)
    _compare(x, w, None, None, act, g)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_float32_bias_beside_16_bit_products(dtype):
    x, w, b, res, g = _inputs(40, 72, 56, dtype, bias=torch.float32)
    _compare(x, w, b, res, "gelu", g)
    assert _step(x, w, b, res, "gelu", g)[1][2].dtype == torch.float32


@gpu
@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views(dtype, m):
    x, w, b, res, g = _inputs(m, 192, 160, dtype)
    pad = lambda t, lead, tail: torch.nn.functional.pad(t, (lead, tail), value=float("nan"))  # noqa: E731
    for lead, tail in ((0, 8), (8, 0), (1, 0), (3, 6)):  # in place, or not aligned
        cut = lambda t: pad(t, lead, tail)[:, lead:lead + t.shape[1]]  # noqa: B023, E731
        _compare(cut(x), cut(w), b, cut(res), "silu", cut(g))
    _compare(x, w.t().contiguous().t(), b, res.t().contiguous().t(), None, g.t().contiguous().t())
    _compare(x[:1].expand(m, -1), w, b, res[:1].expand(m, -1), "relu", g[:1, :1].expand(m, 160))
    _compare(x, w[:1].expand(160, -1), b[:1].expand(160), res, None, g)
    streams = torch.stack((x, x + 1, x - 1), 1)
    _compare(streams, w, b, None, "gelu", torch.stack((g, g, -g), 1))
    _compare(streams[:, 1], w, b, None, "gelu", g)
    if dtype == torch.float32:
        neg = torch.complex(x, x).conj().imag
        assert neg.is_neg()
        _compare(neg, w, b, None, None, g)


@gpu
def test_partial_gradients():
    x, w, b, _, g = _inputs(30, 80, 48, torch.bfloat16)
    _, full = _step(x, w, b, None, "gelu", g)
    for only in range(3):
        leaves = [t.clone() for t in (x, w, b)]
        leaves[only].requires_grad_()
        y = fh.linear(*leaves, activation="gelu")
        (got,) = torch.autograd.grad(y, leaves[only], g)
        assert torch.equal(got, full[only])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [3, 150])
def test_infinity_and_nan_stay_in_their_row(m, dtype):
    x, w, b, _, _ = _inputs(m, 96, 64, dtype)
    w = torch.where(w == 0, torch.ones_like(w), w)
    x[1, 5], x[2, 6] = float("inf"), float("nan")
    y = fh.linear(x, w, b)
    good = [i for i in range(m) if i not in (1, 2)]
    assert y[2].isnan().all() and y[good].isfinite().all()
    assert torch.equal(y[1], torch.copysign(torch.full_like(y[1], float("inf")), w[:, 5]))
    w[7] = 0
    w[7, 5] = float("-inf")
    y = fh.linear(x, w, b)
    assert y[1, 7] == float("-inf") and y[good, 7].isinf().all()
    other = [i for i in range(64) if i != 7]
    assert y[good][:, other].isfinite().all()


@gpu
@pytest.mark.parametrize("act", ACTS[1:])
def test_sums_beyond_half_precision(act):
    """Sums beyond FP16's range beside bf16 results: slopes of 0 and 1, no infinity."""
    x, w, b, _, g = _inputs(20, 64, 40, torch.bfloat16)
    x = x * 1e6
    _, (dx, dw, db, _) = _step(x, w, b, None, act, g)
    want, bound = _formula(x, w, b, None, "relu", g)
    for got, i in ((dx, 1), (dw, 2), (db, 3)):
        assert got.isfinite().all()
        _check(got, want[i], bound[i] + 1e-3 * want[i].abs().max(), act)


@gpu
def test_large_and_small_float32_values():
    x, w, b, _, g = _inputs(40, 64, 48, torch.float32)
    _compare(x * 1e18, w * 1e18, b, None, None, g * 1e-18)
    _compare(x * 1e-16, w * 1e-16, None, None, None, g)


@gpu
def test_no_rows():
    x, w, b, res, g = _inputs(0, 24, 16, torch.bfloat16)
    y, (dx, dw, db, _) = _step(x, w, b, res, "silu", g)
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not dw.any() and not db.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(2, 4096, 100), (400, 3000, 16), (700, 320, 400)])
def test_results_are_the_same_bits_again(m, k, n, dtype):
    x, w, b, res, g = _inputs(m, k, n, dtype)
    first, again = (_step(x, w, b, res, "gelu", g) for _ in range(2))
    assert torch.equal(first[0], again[0]) and all(map(torch.equal, first[1], again[1]))


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """Central differences of sum(g y) in FP32, h = 2^-7: h^2 / 6 times the third derivative (below 4
    a unit of x or w of size about 1) and u / h a term stay below 1% of the gradient's norm."""
    x, w, b, _, g = _inputs(6, 24, 10, torch.float32, seed=11)
    if act == "relu":
        # Sums this far from the step stay on their side of it.
        z = x @ w.t() + b
        g = torch.where(z.abs() < 0.2, torch.zeros_like(g), g)
    _, grads = _step(x, w, b, None, act, g)
    for i, (t, d) in enumerate(zip((x, w, b), grads)):
        v = torch.randn(t.shape, device="cuda")
        h = 2.0**-7
        args = [x, w, b]
        value = []
        for sign in (1, -1):
            args[i] = t + sign * h * v
            value.append((fh.linear(*args, activation=act).double() * g.double()).sum())
        want = (d.double() * v.double()).sum()
        assert abs((value[0] - value[1]) / (2 * h) - want) <= 1e-2 * d.double().norm() * v.double().norm() / t.numel()**0.5


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_second_derivatives_go_native(act):
    x, w, b, _, g = _inputs(4, 12, 9, torch.float32)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    native = {None: lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
              "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[act]

    def grads(f):
        dx, dw, db = torch.autograd.grad(f(x, w, b), (x, w, b), g, create_graph=True)
        return dx, dw, db, *torch.autograd.grad((dx.square().sum() + dw.square().sum()) + db.square().sum(), (x, w),)

    got = grads(lambda *a: fh.linear(*a, activation=act))
    for a, e in zip(got, grads(lambda xx, ww, bb: native(torch.nn.functional.linear(xx, ww, bb)))):
        torch.testing.assert_close(a, e, rtol=1e-3, atol=1e-3)


@gpu
def test_compiled_step_matches():
    x, w, b, res, g = _inputs(33, 72, 40, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
    f = lambda a, ww, bb, r: fh.linear(a, ww, bb, activation="gelu", residual=r)  # noqa: E731
    y = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)
    got = torch.autograd.grad(y, leaves, g)
    want_y, want = _step(x, w, b, res, "gelu", g)
    assert torch.equal(y, want_y) and all(map(torch.equal, got, want))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_cpu_tensors_go_native(dtype, act):
    x, w, b, res, g = _inputs(5, 33, 21, dtype, device="cpu")
    y = fh.linear(x, w, b, activation=act, residual=res)
    want, bound = _formula(x, w, b, res, act, g)
    _check(y, want[0], bound[0], "y")


def test_refusals_on_the_cpu():
    x, w, b, res, _ = _inputs(4, 10, 6, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="unknown activation"):
        fh.linear(x, w, b, activation="swish")
    with pytest.raises(ValueError, match="residual"):
        fh.linear(x, w, b, residual=res[:1])
    with pytest.raises(RuntimeError):
        fh.linear(x, w[:, :9], b)


@gpu
def test_refusals():
    x, w, b, res, g = _inputs(4, 10, 6, torch.bfloat16)
    for args, residual, match in (((x, w[:, :9], b), None, "weight"), ((x, w.float(), b), None, "weight"),
                                  ((x, w, b[:5]), None, "bias"), ((x, w, b.half()), None, "bias"),
                                  ((x, w, b), res[:1], "residual"), ((x, w, b), res.float(), "residual"),
                                  ((x, w.cpu(), b), None, None)):
        with pytest.raises(RuntimeError, match=match):
            fh.linear(*args, residual=residual)
    ops = torch.ops.flash_hypercons
    with pytest.raises(RuntimeError, match="activation"):
        ops._linear(x, w, b, None, 9)
    y, saved = ops._linear_forward(x, w, b, None, 2)
    with pytest.raises(RuntimeError, match="saved"):
        ops._linear_backward(g, x, w, b, saved.float(), 2, True, True, True)
    with pytest.raises(RuntimeError, match="grad"):
        ops._linear_backward(g[:2], x, w, b, saved, 2, True, True, True)
