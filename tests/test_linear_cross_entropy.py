"""linear_cross_entropy and its gradients against their formulas in 64 bits, elementwise.

Bounds: u = 2^-24.  A logit, a sum of K products, is off by at most (K + 8) u sum|x w| (any order, FP32
accumulators); FP32 operands, multiplied as sums of bf16 parts with the products below 2^-22 left out, by
(2 K + 16) u sum|x w|; the bias adds 2 u |z|.  An exponential of d errs by (2 |d| + 4) u of itself, through
its argument's rounding and the hardware's last place; it is scaled twice more on its way into the row's
sum, by the 64 logits' maximum and by the row's.  That sum is added in runs of at most V / 64 + 64 terms.
A logarithm errs by 4 u of itself and its argument's relative error.  So lse errs by

    the largest error of the row's logits + sum over v of p_v (4 |z_v - max| + 8) u + (V / 64 + 64) u
    + 4 u |lse - max| + 2 u |lse|,

the loss by that, the target's logit's error and 2 u of its size, and p_v = exp(z_v - lse) by the errors of
z_v and lse and (2 |z_v - lse| + 4) u relatively (times 1.1 for what is not of first order).  dz is rounded
to the storage type (half an ulp; FP16 through a scale, with steps of 2^-39 of the largest factor), and
the sums over V and T err like the logits' over K.  What lies below 2^-126, the smallest normal FP32 number,
may count as zero: the hardware's exponential gives none below it, and the matrix instructions take none in (an
FP32 operand's last bf16 part lies up to 2^-16 below the operand) nor give one out: 2^-125 for each p, dz and
product.  The results' own storage type adds half an ulp, and half a subnormal step; beyond its range they
are infinite.

Where the gradients are formed with the loss, 16-bit operands' exponentials beside the maximum of their 64 are
kept in FP16 times 2^15: off by 2^-11 of themselves and 2^-40, except the target's.  FP16's dz is then kept
in steps of 2^-40.  Every test below that compares with the formula takes both ways.
"""

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp

U = 2.0**-24
TINY = 2.0**-125
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
REDUCTIONS = ["mean", "sum", "none"]
gpu = pytest.mark.gpu


def _sum_error(k, dtype):
    return ((2 * k + 16) if dtype == torch.float32 else (k + 8)) * U


def _formula(x, w, targets, b, reduction, g, ignore=-100, ahead=False):
    """loss, dx, dw, db in 64 bits and their bounds, for targets in range or ignored."""
    dtype, dev = x.dtype, x.device
    k, vocab = x.shape[-1], w.shape[0]
    t = targets.reshape(-1).long()
    here = t != ignore
    xd = torch.where(here[:, None], x.double().reshape(-1, k), 0.0)
    wd = w.double()
    rows = len(t)
    count = int(here.sum())
    f = (g.double().reshape(-1) if reduction == "none" else g.double().expand(rows)) * here
    if reduction == "mean" and count:
        f = f / count
    most = f[f.isfinite()].abs().max() if rows else torch.zeros((), device=dev)
    losses, el = (torch.zeros(rows, dtype=torch.float64, device=dev) for _ in range(2))
    dx, edx = torch.zeros_like(xd), torch.zeros_like(xd)
    dw, edw = torch.zeros_like(wd), torch.zeros_like(wd)
    db, edb = (torch.zeros(vocab, dtype=torch.float64, device=dev) for _ in range(2))
    step = max(1, (1 << 26) // vocab)
    for i in range(0, rows, step):
        s = slice(i, i + step)
        at = t[s].clamp(min=0)[:, None]
        z = xd[s] @ wd.t()
        ez = _sum_error(k, dtype) * (xd[s].abs() @ wd.abs().t())
        if b is not None:
            z = z + b.double()
            ez = ez + 2 * U * z.abs().nan_to_num(0, 0, 0)
        top = z.amax(1, keepdim=True)
        lse = torch.logsumexp(z, 1, keepdim=True)
        p = (z - lse).exp()
        far = (z - top).abs().nan_to_num(0, 0, 0)
        elz = (ez.amax(1, keepdim=True) + (p * (4 * far + 8)).sum(1, keepdim=True) * U + (vocab / 64 + 64) * U
               + 4 * U * (lse - top).abs() + 2 * U * lse.abs())
        zt = z.gather(1, at)
        losses[s] = torch.where(here[s], (lse - zt).squeeze(1), 0.0)
        el[s] = torch.where(here[s], (elz + ez.gather(1, at) + 2 * U * (lse - zt).abs()).squeeze(1), 0.0)
        ep = 1.1 * p * (ez + elz + (2 * far + 2 * (top - lse).abs() + 4) * U)
        hot = torch.zeros_like(p).scatter_(1, at, 1.0)
        if ahead and dtype != torch.float32:
            ep = ep + (1 - hot) * (2.0**-11 * p * (1 + 1.1 * U) + 2.0**-40 + 2.0**-11 * ep)
        dz = (p - hot) * f[s, None]
        edz = (ep + 2 * U * hot + TINY) * f[s, None].abs() + 2 * U * dz.abs() + TINY * (f[s, None] != 0)
        edz = edz + half_ulp(dtype) * (dz.abs() + edz) + (2.0**-39 * most if dtype == torch.float16 else floor(dtype)) * (f[s, None] != 0)
        size = dz.abs() + edz
        dx[s] = dz @ wd
        edx[s] = edz @ wd.abs() + _sum_error(vocab, dtype) * (size @ wd.abs()) + vocab * TINY
        dw += dz.t() @ xd[s]
        edw += edz.t() @ xd[s].abs() + _sum_error(rows, dtype) * (size.t() @ xd[s].abs()) + len(z) * TINY
        db += dz.sum(0)
        edb += edz.sum(0) + (rows + 8) * U * size.sum(0)
    if reduction == "none":
        loss, eloss = losses.reshape(targets.shape), el.reshape(targets.shape)
    else:
        scale = 1 if reduction == "sum" else count  # the mean of none is NaN
        loss, eloss = losses.sum() / scale, el.sum() / scale + 2 * U * losses.sum().abs() / scale
    return (loss, dx.reshape(x.shape), dw, db), (eloss, edx.reshape(x.shape), edw, edb)


def _check(got, want, bound, what):
    dt = got.dtype
    got = got.detach().double()
    assert got.shape == want.shape, what
    limit = half_ulp(dt) * want.abs() + (1 + half_ulp(dt)) * bound + floor(dt) + (U * want.abs() if dt == torch.float32 else 0)
    off = (got - want).abs()
    good = (off <= limit) | (got.isnan() & want.isnan())
    good |= got.isinf() & (want.sign() == got.sign()) & (want.abs() + limit > torch.finfo(dt).max)
    assert bool(good.all()), f"{what}: {(off / limit).nan_to_num(9e9).max().item():.2f} times the bound"


OPS = torch.ops.flash_hypercons


def _step(x, w, targets, b, reduction, g, way=None, **args):
    """Loss and gradients: by autograd, or by the operators of one way of forming them."""
    if way is None:
        leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
        loss = fh.linear_cross_entropy(leaves[0], leaves[1], targets, leaves[2], reduction=reduction, **args)
        grads = list(torch.autograd.grad(loss, [t for t in leaves if t is not None], g))
        return [loss.detach(), *grads]
    how = args.get("ignore_index", -100), {"none": 0, "sum": 1, "mean": 2}[reduction]
    wanted = True, True, b is not None
    if way == "ahead":
        loss, *sums = OPS._linear_cross_entropy_ahead(x, w, targets, b, *how, *wanted)
        grads = OPS._linear_cross_entropy_scale(g, x, w, targets, b, *sums, *how)
    else:
        loss, lse = OPS._linear_cross_entropy_forward(x, w, targets, b, *how)
        grads = OPS._linear_cross_entropy_backward(g, x, w, targets, b, lse, *how, *wanted)
    return [loss, *grads[: 2 + (b is not None)]]


def _ways(reduction):
    return ["again"] if reduction == "none" else ["again", "ahead"]


def _compare(x, w, targets, b=None, reduction="mean", g=None, **args):
    if g is None:
        g = torch.rand(targets.shape, device=x.device) if reduction == "none" else torch.tensor(3.0, device=x.device)
    default = _step(x, w, targets, b, reduction, g, **args)
    found = []
    for way in _ways(reduction):
        got = _step(x, w, targets, b, reduction, g, way, **args)
        want, bound = _formula(x, w, targets, b, reduction, g, args.get("ignore_index", -100), way == "ahead")
        assert got[0].dtype == torch.float32
        for name, a, e, limit in zip(("loss", "dx", "dw", "db"), got, want, bound):
            _check(a, e, limit, f"{way} {name}")
        found.append(all(torch.equal(a.nan_to_num(7e7), e.nan_to_num(7e7)) for a, e in zip(default, got)))
    rows = targets.numel()
    ahead = reduction != "none" and rows >= (128 if x.dtype == torch.float32 else 1024)
    assert found[ahead]  # what autograd takes
    with torch.no_grad():
        again = fh.linear_cross_entropy(x, w, targets, b, reduction=reduction, **args)
    torch.testing.assert_close(again, default[0], rtol=1e-6, atol=0, equal_nan=True)
    return default


def _inputs(m, k, v, dtype, seed=0, device="cuda", ignored=0.0, bias=None, sure=6.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device=device)  # noqa: E731
    w = (normal(v, k) * k**-0.5).to(dtype)
    t = torch.randint(0, v, (m,), generator=gen, device=device)
    x = (normal(m, k) + w[t].float() * sure * torch.rand(m, 1, generator=gen, device=device)).to(dtype)
    if ignored:
        t[torch.rand(m, generator=gen, device=device) < ignored] = -100
    return x, w, t, normal(v).to(bias or dtype)


# Around the edges of vectors, tiles, groups of 64 and slices.
SIZES = [(1, 1, 1), (1, 8, 64), (3, 7, 5), (2, 64, 33), (40, 16, 20), (33, 72, 32), (31, 128, 65), (1, 4096, 1000),
         (32, 40, 3000), (64, 200, 1000), (65, 264, 129), (130, 72, 4100), (257, 100, 513), (300, 2056, 300),
         (513, 520, 264), (1000, 16, 2000), (2000, 96, 31), (40, 64, 30011), (1100, 203, 5000), (2100, 96, 9001)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,v", SIZES)
def test_sizes(m, k, v, dtype):
    x, w, t, b = _inputs(m, k, v, dtype, seed=m + k + v, ignored=0.2 * (m % 3))
    _compare(x, w, t, b if (m + v) % 2 else None, REDUCTIONS[(m + k) % 3])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("reduction", REDUCTIONS)
@pytest.mark.parametrize("m", [1, 20, 150, 700])
def test_reductions(m, reduction, dtype):
    x, w, t, b = _inputs(m, 136, 777, dtype, seed=m)
    _compare(x, w, t, b, reduction)
    t[m // 2:] = -100
    if m > 1:
        _compare(x, w, t, None, reduction)


@gpu
@pytest.mark.parametrize("way", ["again", "ahead"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [1, 90, 600])
def test_positions_without_a_target_take_no_part(m, dtype, way):
    x, w, t, b = _inputs(m + 40, 72, 500, dtype, seed=m)
    t[5:45] = -1
    x[5:45] = float("nan")
    x[20] = float("inf")
    keep = torch.ones(m + 40, dtype=torch.bool, device="cuda")
    keep[5:45] = t[m + 1:m + 1] = False
    for reduction in (r for r in REDUCTIONS if way in _ways(r)):
        g = torch.rand(m + 40, device="cuda") if reduction == "none" else torch.tensor(1.0, device="cuda")
        got = _step(x, w, t, b, reduction, g, way, ignore_index=-1)
        assert not got[1][5:45].any()
        if reduction == "none":
            assert not got[0][5:45].any()
        # As the formula of the others alone, whose bounds hold whatever slices and parts their number goes in.
        want, bound = _formula(x[keep], w, t[keep], b, reduction, g[keep] if reduction == "none" else g, -1, way == "ahead")
        found = got[0][keep] if reduction == "none" else got[0], got[1][keep], *got[2:]
        for name, a, e, limit in zip(("loss", "dx", "dw", "db"), found, want, bound):
            _check(a, e, limit, name)


@gpu
@pytest.mark.parametrize("way", ["again", "ahead"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [1, 300])
def test_no_target_at_all(m, dtype, way):
    x, w, t, b = _inputs(m, 40, 100, dtype)
    t[:] = -100
    for reduction in (r for r in REDUCTIONS if way in _ways(r)):
        g = torch.ones(m if reduction == "none" else (), device="cuda")
        loss, *grads = _step(x, w, t, b, reduction, g, way)
        assert loss.isnan().all() if reduction == "mean" else not loss.any()
        assert not any(d.any() for d in grads)


@gpu
def test_no_positions():
    x, w, t, b = _inputs(0, 24, 16, torch.bfloat16)
    for reduction in REDUCTIONS:
        loss, dx, dw, db = _step(x, w, t, b, reduction, torch.ones(0 if reduction == "none" else (), device="cuda"))
        assert loss.shape == ((0,) if reduction == "none" else ()) and (reduction != "mean" or loss.isnan())
        assert dx.shape == (0, 24) and not dw.any() and not db.any()


@gpu
@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_targets_out_of_range(m, dtype):
    x, w, t, _ = _inputs(m, 40, 100, dtype)
    t[1], t[2] = 100, -7
    g = torch.ones(m, device="cuda")
    loss, dx, dw = _step(x, w, t, None, "none", g)
    good = [i for i in range(m) if i not in (1, 2)]
    assert loss[[1, 2]].isnan().all() and loss[good].isfinite().all()
    assert dx[[1, 2]].isnan().all() and dx[good].isfinite().all() and dw.isnan().all()
    assert fh.linear_cross_entropy(x, w, t).isnan()
    loss, dx, dw = _step(x, w, t, None, "sum", g[0], "ahead")
    assert loss.isnan() and dx[[1, 2]].isnan().all() and dx[good].isfinite().all() and dw.isnan().all()


@gpu
@pytest.mark.parametrize("way", ["again", "ahead"])
@pytest.mark.parametrize("m", [2, 150])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_words_that_a_bias_rules_out(m, dtype, way):
    """A bias of -inf or of the type's lowest value, as a padded vocabulary has."""
    x, w, t, b = _inputs(m, 64, 300, dtype)
    t = t % 200
    for low in (float("-inf"), torch.finfo(dtype).min):
        b[200:] = low
        got = _step(x, w, t, b, "mean", torch.tensor(1.0, device="cuda"), way)
        want, bound = _formula(x, w[:200], t, b[:200], "mean", torch.tensor(1.0, device="cuda"), ahead=way == "ahead")
        _check(got[0], want[0], bound[0], "loss")
        _check(got[1], want[1], bound[1], "dx")
        _check(got[2][:200], want[2], bound[2], "dw")
        assert not got[2][200:].any() and not got[3][200:].any()
    b[:] = float("-inf")  # nothing is left
    assert _step(x, w, t, b, "none", torch.ones(m, device="cuda"))[0].isnan().all()
    b[:] = 0
    b[t[0]] = float("-inf")  # the target is ruled out
    assert _step(x, w, t, b, "none", torch.ones(m, device="cuda"))[0][0] == float("inf")


@gpu
@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_infinity_and_nan_stay_in_their_row(m, dtype):
    x, w, t, _ = _inputs(m, 96, 64, dtype)
    x[1, 5], x[2, 6] = float("inf"), float("nan")
    loss, dx, _ = _step(x, w, t, None, "none", torch.ones(m, device="cuda"))
    good = [i for i in range(m) if i not in (1, 2)]
    assert loss[[1, 2]].isnan().all() and loss[good].isfinite().all() and dx[good].isfinite().all()
    loss, dx, _ = _step(x, w, t, None, "sum", torch.tensor(1.0, device="cuda"), "ahead")
    assert loss.isnan() and dx[[1, 2]].isnan().all() and dx[good].isfinite().all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_large_logits(dtype):
    """Logits far beyond exp's range, certain and hopeless targets."""
    x, w, t, _ = _inputs(100, 64, 200, dtype, sure=0.0)
    for reduction in ("none", "sum"):
        _compare(x * 60, w * 4, t, None, reduction)
        _compare(x * 60, w * 4, (x.float() @ w.float().t()).argmax(1), None, reduction)


@gpu
@pytest.mark.parametrize("scale", [1e-6, 1.0, 65536.0, 1e20])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_upstream_gradients_of_any_size(dtype, scale):
    x, w, t, b = _inputs(80, 64, 3000, dtype)
    if dtype == torch.float16:
        scale = min(scale, 65536.0)
    _compare(x, w, t, b, "mean", torch.tensor(scale, device="cuda"))
    g = torch.randn(80, device="cuda") * 10.0 ** torch.linspace(-6, 0, 80, device="cuda") * scale
    g[7] = 0
    _compare(x, w, t, b, "none", g)


@gpu
def test_zero_and_infinite_upstream_gradients():
    x, w, t, b = _inputs(40, 64, 300, torch.float16)
    for way in _ways("mean"):
        assert not any(d.any() for d in _step(x, w, t, b, "mean", torch.tensor(0.0, device="cuda"), way)[1:])
        for bad in (float("inf"), float("nan")):
            grads = _step(x, w, t, b, "mean", torch.tensor(bad, device="cuda"), way)[1:]
            assert all(not d.isfinite().all() for d in grads)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_float32_bias_beside_16_bit_products(dtype):
    x, w, t, b = _inputs(70, 72, 560, dtype, bias=torch.float32)
    assert _compare(x, w, t, b)[3].dtype == torch.float32


@gpu
@pytest.mark.parametrize("m", [6, 210])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views(dtype, m):
    x, w, t, b = _inputs(m, 192, 360, dtype)
    pad = lambda a, lead, tail: torch.nn.functional.pad(a, (lead, tail), value=float("nan"))  # noqa: E731
    for lead, tail in ((0, 8), (8, 0), (1, 0), (3, 6)):
        cut = lambda a: pad(a, lead, tail)[:, lead:lead + a.shape[1]]  # noqa: B023, E731
        _compare(cut(x), cut(w), t, b)
    _compare(x, w.t().contiguous().t(), t.int(), b)
    _compare(x[:1].expand(m, -1), w, t, b[:1].expand(360), "sum")
    streams = torch.stack((x, x + 1, x - 1), 1)
    _compare(streams[:, 1], w, t)
    three = streams.reshape(m // 3, 3, 3, 192)
    _compare(three[:, :, 0], w, t.view(m // 3, 3), b, "none", torch.rand(3, m // 3, device="cuda").t())
    _compare(x, w, t, None, "none", torch.ones(1, device="cuda").expand(m))
    _compare(x[0], w, t[0], b, "none", torch.tensor(0.5, device="cuda"))


@gpu
@pytest.mark.parametrize("m", [50, 1300])
def test_partial_gradients(m):
    x, w, t, b = _inputs(m, 80, 1000, torch.bfloat16, ignored=0.3)
    g = torch.tensor(2.0, device="cuda")
    full = _step(x, w, t, b, "mean", g)[1:]
    for only in range(3):
        leaves = [a.clone() for a in (x, w, b)]
        leaves[only].requires_grad_()
        loss = fh.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        assert torch.equal(torch.autograd.grad(loss, leaves[only], g)[0], full[only])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,v", [(2, 4096, 1000), (400, 512, 3000), (700, 72, 20), (1500, 256, 4000)])
def test_results_are_the_same_bits_again(m, k, v, dtype):
    x, w, t, b = _inputs(m, k, v, dtype, ignored=0.2)
    g = torch.tensor(1.0, device="cuda")
    first, again = (_step(x, w, t, b, "mean", g) for _ in range(2))
    assert all(map(torch.equal, first, again))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_a_long_batch_over_many_words(dtype):
    """More rows, logits and statistics than the kernels take at a time."""
    x, w, t, b = _inputs(66000, 8, 33000, dtype, ignored=0.001)
    _compare(x, w, t, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_millions_of_rows(dtype):
    """More rows than a grid's second dimension has blocks of 64."""
    x, w, t, b = _inputs(4_300_000, 8, 9, dtype, ignored=0.1)
    _compare(x, w, t, b)


@gpu
@pytest.mark.parametrize("m", [5, 300, 1100])
def test_a_weight_beyond_two_billion_elements(m):
    """Offsets past 2^31 elements: the loss, dx and some rows of dW against FP32 products, to FP32 and bf16 rounding."""
    k, v = 17000, 131072
    gen = torch.Generator(device="cuda").manual_seed(m)
    w = torch.randn(v, k, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(k**-0.5)
    t = torch.randint(0, v, (m,), generator=gen, device="cuda")
    t[0], t[1] = v - 1, 0
    x = torch.randn(m, k, generator=gen, device="cuda").add_(5 * w[t].float()).bfloat16()
    loss, dx, dw = _step(x, w, t, None, "mean", torch.tensor(float(m), device="cuda"))
    z = torch.cat([x.float() @ w[i:i + 16384].float().t() for i in range(0, v, 16384)], 1)
    torch.testing.assert_close(loss, torch.nn.functional.cross_entropy(z, t), rtol=1e-5, atol=1e-5)
    dz = z.softmax(1)
    dz[torch.arange(m), t] -= 1
    want = sum(dz[:, i:i + 16384] @ w[i:i + 16384].float() for i in range(0, v, 16384))
    assert (dx.float() - want).norm() <= 6e-3 * want.norm()
    rows = torch.tensor([0, 1, 63, 126322, 126323, 126400, v - 2, v - 1], device="cuda")  # 2^31 / k = 126322.6
    want = dz[:, rows].t() @ x.float()
    assert ((dw[rows].float() - want).norm(dim=1) <= 6e-3 * want.norm(dim=1)).all()


@gpu
def test_gradients_against_differences():
    """Central differences in FP32 at h = 2^-6: the third derivatives' h^2 / 6 and u / h a logit stay below 1%."""
    x, w, t, b = _inputs(6, 24, 40, torch.float32, seed=11, ignored=0.2)
    grads = _step(x, w, t, b, "sum", torch.tensor(1.0, device="cuda"))[1:]
    for i, d in enumerate(grads):
        v = torch.randn(d.shape, device="cuda")
        v = v / v.norm()
        args, value = [x, w, b], []
        for sign in (1, -1):
            args[i] = (x, w, b)[i] + sign * 2.0**-6 * v
            value.append(fh.linear_cross_entropy(args[0], args[1], t, args[2], reduction="none").double().sum())
        want = (d.double() * v.double()).sum()
        assert abs((value[0] - value[1]) / 2.0**-5 - want) <= 1e-2 * d.double().norm()


@gpu
@pytest.mark.parametrize("m", [7, 140])  # of the gradients formed again, and with the loss
@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_second_derivatives_go_native(reduction, m):
    x, w, t, b = _inputs(m, 12, 9, torch.float32, ignored=0.3)
    x, w, b = (a.requires_grad_() for a in (x, w, b))
    g = torch.rand(m if reduction == "none" else (), device="cuda")

    def grads(loss):
        d = torch.autograd.grad(loss, (x, w, b), g, create_graph=True)
        return *d, *torch.autograd.grad(sum(a.square().sum() for a in d), (x, w, b))

    got = grads(fh.linear_cross_entropy(x, w, t, b, reduction=reduction))
    native = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b), t, reduction=reduction)
    for a, e in zip(got, grads(native)):
        torch.testing.assert_close(a, e, rtol=1e-4, atol=1e-5)


@gpu
def test_function_transforms_and_tangents_go_native():
    x, w, t, _ = _inputs(6, 12, 9, torch.float32)
    loss = lambda a, b: fh.linear_cross_entropy(a, b, t)  # noqa: E731
    native = lambda a, b: torch.nn.functional.cross_entropy(a @ b.t(), t)  # noqa: E731
    torch.testing.assert_close(torch.func.grad(loss, (0, 1))(x, w), torch.func.grad(native, (0, 1))(x, w))
    for a, e in zip(torch.func.jvp(loss, (x, w), (w[:6], w + 1)), torch.func.jvp(native, (x, w), (w[:6], w + 1))):
        torch.testing.assert_close(a, e)
    many = torch.func.vmap(lambda a: fh.linear_cross_entropy(a, w, t, reduction="sum"))(torch.stack((x, x + 1)))
    torch.testing.assert_close(many[1], fh.linear_cross_entropy(x + 1, w, t, reduction="sum"))


@gpu
def test_a_graph_that_is_walked_twice():
    x, w, t, b = _inputs(1300, 80, 500, torch.bfloat16)
    leaves = [a.clone().requires_grad_() for a in (x, w, b)]
    loss = fh.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    for g in (1.0, 0.125):
        g = torch.tensor(g, device="cuda")
        got = torch.autograd.grad(loss, leaves, g, retain_graph=True)
        assert all(map(torch.equal, got, _step(x, w, t, b, "mean", g)[1:]))


@gpu
def test_compiled_step_matches():
    f = torch.compile(lambda a, ww, tt, bb: fh.linear_cross_entropy(a, ww, tt, bb), fullgraph=True, backend="aot_eager")
    g = torch.tensor(1.0, device="cuda")
    for m, v in ((33, 400), (40, 401), (1300, 500), (1400, 700)):  # sizes become symbols; both ways
        x, w, t, b = _inputs(m, 72, v, torch.bfloat16)
        leaves = [a.clone().requires_grad_() for a in (x, w, b)]
        loss = f(leaves[0], leaves[1], t, leaves[2])
        got = [loss.detach(), *torch.autograd.grad(loss, leaves, g)]
        assert all(map(torch.equal, got, _step(x, w, t, b, "mean", g)))


@pytest.mark.parametrize("reduction", REDUCTIONS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_cpu_tensors_go_native(dtype, reduction):
    x, w, t, b = _inputs(9, 33, 21, dtype, device="cpu", ignored=0.3)
    x[t == -100] = float("nan")
    g = torch.rand(9) if reduction == "none" else torch.tensor(1.0)
    got = _step(x, w, t, b, reduction, g)
    want, bound = _formula(x, w, t, b, reduction, g)
    for a, e, limit in zip(got, want, bound):
        _check(a, e, limit, reduction)


def test_refusals_on_the_cpu():
    x, w, t, b = _inputs(4, 10, 6, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="reduction"):
        fh.linear_cross_entropy(x, w, t, b, reduction="max")
    with pytest.raises(ValueError, match="targets"):
        fh.linear_cross_entropy(x, w, t[:3], b)
    with pytest.raises(RuntimeError):
        fh.linear_cross_entropy(x, w[:, :9], t, b)
    with pytest.raises(IndexError):
        fh.linear_cross_entropy(x, w, t + 6, b)


@gpu
def test_refusals():
    x, w, t, b = _inputs(4, 10, 6, torch.bfloat16)
    for args, match in (((x, w[:, :9], t, b), "weight"), ((x, w.float(), t, b), "weight"), ((x, w, t, b[:5]), "bias"),
                        ((x, w, t, b.half()), "bias"), ((x, w, t[:3], b), "targets"), ((x, w.cpu(), t, b), None)):
        with pytest.raises(RuntimeError, match=match):
            fh.linear_cross_entropy(*args)
    ops = torch.ops.flash_hypercons
    with pytest.raises(RuntimeError, match="reduction"):
        ops._linear_cross_entropy(x, w, t, b, -100, 3)
    with pytest.raises(RuntimeError, match="targets"):
        ops._linear_cross_entropy(x, w, t.float(), b, -100, 2)
    loss, lse = ops._linear_cross_entropy_forward(x, w, t, b, -100, 2)
    with pytest.raises(RuntimeError, match="sums"):
        ops._linear_cross_entropy_backward(loss, x, w, t, b, lse.half(), -100, 2, True, True, True)
    with pytest.raises(RuntimeError, match="grad"):
        ops._linear_cross_entropy_backward(lse, x, w, t, b, lse, -100, 2, True, True, True)
    with pytest.raises(RuntimeError, match="sum or mean"):
        ops._linear_cross_entropy_ahead(x, w, t, b, -100, 0, True, True, True)
    loss, *sums = ops._linear_cross_entropy_ahead(x, w, t, b, -100, 2, True, True, False)
    assert [a.numel() for a in sums] == [5, 40, 60, 0]
    with pytest.raises(RuntimeError, match="sums"):
        ops._linear_cross_entropy_scale(loss, x, w, t, b, sums[0], sums[1][:2], *sums[2:], -100, 2)
    with pytest.raises(RuntimeError, match="sums"):
        ops._linear_cross_entropy_scale(loss, x, w, t, b, sums[0][:0], *sums[1:], -100, 2)
    with pytest.raises(RuntimeError, match="grad"):
        ops._linear_cross_entropy_scale(lse, x, w, t, b, *sums, -100, 2)
