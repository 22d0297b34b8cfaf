"""embedding and its gradient against their formulas in 64 bits, elementwise.

Bounds: u = 2^-24.  scale is rounded to FP32 and multiplied once: 2 u of the result.  A sum of n terms
in FP32 is off by at most n u times the sum of their sizes, in any order.  The storage type adds half an
ulp of the result, and half a subnormal step.
"""

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp

U = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def _check(got, want, bound, what):
    dt = got.dtype
    got = got.detach().double().cpu()
    limit = half_ulp(dt) * want.abs() + (1 + half_ulp(dt)) * bound + floor(dt)
    off = (got - want).abs()
    assert got.shape == want.shape
    assert bool((off <= limit).all()), f"{what}: {(off / limit).nan_to_num(0).max().item():.2f} times the bound"


def _formula(tokens, weight, g, scale, streams, padding):
    """y, dweight and their bounds."""
    t, w = tokens.cpu().long(), weight.double().cpu()
    y = w[t] * scale
    if streams:
        y = y.unsqueeze(-2).expand(*t.shape, streams, w.shape[1])
    rows = g.double().cpu().reshape(t.numel(), max(1, streams or 0), w.shape[1])
    flat = t.reshape(-1)
    keep = (flat != (-1 if padding is None else padding)).double()
    dw = torch.zeros_like(w).index_add_(0, flat, rows.sum(1) * keep[:, None]) * scale
    size = torch.zeros_like(w).index_add_(0, flat, rows.abs().sum(1) * keep[:, None]) * abs(scale)
    terms = torch.bincount(flat, minlength=len(w)).double()[:, None] * max(1, streams or 0)
    return (y, dw), (2 * U * y.abs(), (terms + 2) * U * size)


def _step(tokens, weight, g, **args):
    leaf = weight.detach().requires_grad_()
    y = fh.embedding(tokens, leaf, **args)
    (dw,) = torch.autograd.grad(y, leaf, g)
    return y.detach(), dw


def _compare(tokens, weight, g, scale=1.0, streams=None, padding=None):
    y, dw = _step(tokens, weight, g, scale=scale, streams=streams, padding_idx=padding)
    want, bound = _formula(tokens, weight, g, scale, streams, padding)
    assert y.dtype == dw.dtype == weight.dtype and y.is_contiguous() and dw.is_contiguous()
    _check(y, want[0], bound[0], "y")
    _check(dw, want[1], bound[1], "dw")
    with torch.no_grad():
        assert torch.equal(fh.embedding(tokens, weight, scale=scale, streams=streams, padding_idx=padding), y)
    if scale == 1.0:
        assert torch.equal(y.double().cpu(), want[0])  # copies


def _inputs(shape, cols, vocab, dtype, streams=None, seed=0, device="cuda", hot=0.3):
    """Tokens of which about a share `hot` are one, the rest spread over the vocabulary."""
    gen = torch.Generator(device=device).manual_seed(seed)
    shape = (shape,) if isinstance(shape, int) else shape
    tokens = torch.randint(0, vocab, shape, generator=gen, device=device)
    tokens[torch.rand(shape, generator=gen, device=device) < hot] = vocab // 2
    normal = lambda *s: torch.randn(s, generator=gen, device=device).to(dtype)  # noqa: E731
    return tokens, normal(vocab, cols), normal(*shape, *((streams,) if streams else ()), cols)


# Around the edges of vectors, strips, chunks, a sort's tiles and digits.
SIZES = [(1, 1, 1), (1, 8, 5), (2, 7, 2), (63, 64, 63), (64, 65, 64), (65, 513, 65), (200, 1027, 511), (1000, 40, 3),
         (1024, 16, 512), (1025, 9, 4095), (4096, 24, 50), (4097, 33, 1000), (16384, 8, 262143), (16385, 8, 20011),
         (40000, 72, 700), (300, 4104, 90)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,cols,vocab", SIZES)
def test_sizes(tokens, cols, vocab, dtype):
    streams = (None, 1, 2, 4, 3)[(tokens + cols) % 5] if tokens * cols < 1 << 21 else None
    t, w, g = _inputs(tokens, cols, vocab, dtype, streams, seed=tokens + cols)
    _compare(t, w, g, 1.0 if cols % 2 else cols**0.5, streams, vocab // 3 if tokens % 2 else None)


@gpu
@pytest.mark.parametrize("hot", [0.0, 0.9, 1.0])
@pytest.mark.parametrize("tokens", [100, 3000, 20000, 70000])
def test_runs_of_any_length(tokens, hot):
    """From every token once to one token alone, over many chunks."""
    t, w, g = _inputs(tokens, 40, 5000, torch.float32, seed=tokens, hot=hot)
    _compare(t, w, g)
    _compare(t, w, g, padding=2500)  # what is hot has no gradient


@gpu
@pytest.mark.parametrize("tokens", [40, 3000, 5000, 20000, 600000])
def test_vocabularies_of_many_digits(tokens):
    """Three and four passes of a sort, by one workgroup and by several of one, four and sixteen thousand keys."""
    for vocab in (3_000_000, 1 << 27 | 1):
        t = torch.randint(0, vocab, (tokens,), device="cuda")
        t[: tokens // 3] = t[0]
        w = torch.arange(vocab, device="cuda").unsqueeze(1).float()
        g = torch.randint(-8, 9, (tokens, 1), device="cuda").float()  # whole numbers: sums are exact in any order
        y, dw = _step(t, w, g)
        assert torch.equal(y, w[t])
        assert torch.equal(dw, torch.zeros(vocab, 1, device="cuda").index_add_(0, t, g))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_runs_that_end_at_the_borders_of_chunks(dtype):
    for length in (15, 16, 17, 31, 32, 33, 64, 128):
        t = torch.arange(50, device="cuda").repeat_interleave(length)
        t = t[torch.randperm(len(t), device="cuda")]
        g = torch.randn(len(t), 24, device="cuda").to(dtype)
        _compare(t, torch.randn(50, 24, device="cuda").to(dtype), g)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views(dtype):
    t, w, g = _inputs((6, 50), 96, 70, dtype, 2)
    pad = lambda x, lead, tail: torch.nn.functional.pad(x, (lead, tail), value=float("nan"))  # noqa: E731
    for lead, tail in ((0, 8), (1, 0), (3, 6)):
        cut = lambda x: pad(x, lead, tail)[..., lead:lead + x.shape[-1]]  # noqa: B023, E731
        _compare(t, cut(w), cut(g), 2.5, 2)
    _compare(t.int(), w, g, -0.5, 2)
    _compare(t.t(), w, g.transpose(0, 1), 1.0, 2)
    _compare(t[:, ::2], w.t().contiguous().t(), g[:, ::2], 1.0, 2)
    _compare(t, w[:1].expand(70, -1), g[:1, :1, :1].expand(6, 50, 2, 96), 3.0, 2)
    _compare(t[0, 0], w, g[0, 0], 1.0, 2)
    _compare(t.reshape(2, 3, 50), w, g.reshape(2, 3, 50, 2, 96), 1.0, 2)
    if dtype == torch.float32:
        neg = torch.complex(w, w).conj().imag
        assert neg.is_neg()
        _compare(t, neg, torch.complex(g, g).conj().imag, 1.0, 2)


@gpu
def test_no_tokens():
    t, w, g = _inputs(0, 24, 16, torch.bfloat16, 3)
    y, dw = _step(t, w, g, streams=3)
    assert y.shape == (0, 3, 24) and dw.shape == (16, 24) and not dw.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_tokens_out_of_range(dtype):
    t, w, g = _inputs(500, 40, 30, dtype)
    bad = t.clone()
    bad[3], bad[100], bad[499], bad[7] = -1, 30, 2**40, -(2**40)
    y, dw = _step(bad, w, g, scale=2.0)
    at = torch.zeros(500, dtype=torch.bool, device="cuda")
    at[[3, 100, 499, 7]] = True
    assert y[at].isnan().all() and y[~at].isfinite().all()
    assert torch.equal(dw, _step(t[~at], w, g[~at], scale=2.0)[1])


@gpu
def test_infinity_and_nan_stay_in_their_row():
    t, w, g = _inputs(300, 40, 60, torch.bfloat16, hot=0.0)
    w[5], g[t == 9] = float("inf"), float("nan")
    y, dw = _step(t, w, g)
    assert y[t == 5].isinf().all() and y[t != 5].isfinite().all()
    assert dw[9].isnan().all() and dw[[i for i in range(60) if i != 9]].isfinite().all()


@gpu
@pytest.mark.parametrize("tokens", [700, 16384, 50000])
def test_results_are_the_same_bits_again(tokens):
    t, w, g = _inputs(tokens, 72, 900, torch.float32, 2)
    first, again = (_step(t, w, g, streams=2) for _ in range(2))
    assert all(map(torch.equal, first, again))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,cols,vocab", [(0, 5, 300), (1, 3, 32768), (900, 7, 32768), (2048, 130, 32769),
                                              (1711, 1079, 872), (2048, 65, 70001)])
def test_rows_without_a_token_are_zero(tokens, cols, vocab, dtype):
    """Whole blocks, parts and single rows of the table, whose memory held NaN before; padded ones too."""
    t, w, g = _inputs(tokens, cols, vocab, dtype)
    if tokens:
        t[: tokens // 2] = torch.arange(tokens // 2, device="cuda") % vocab  # a dense block
    for padding in (None, 0):
        before = torch.full_like(w, float("nan"))
        del before
        _compare(t, w, g, padding=padding)


@gpu
def test_long_rows_of_a_large_table():
    """Offsets beyond 2^31 elements, in the table, the result and the gradients."""
    w = torch.empty(300000, 8192, dtype=torch.bfloat16, device="cuda")
    t = torch.tensor([299999, 5, 299999, 262144, 0], device="cuda")
    rows = torch.randn(4, 8192, device="cuda").bfloat16()
    w[[299999, 5, 262144, 0]] = rows
    y, dw = _step(t, w, w[t].neg())
    assert torch.equal(y, rows[[0, 1, 0, 2, 3]])
    assert torch.equal(dw[[5, 262144, 0]], -rows[1:]) and torch.equal(dw[299999], -2 * rows[0])
    assert dw.count_nonzero() == rows.count_nonzero()
    del w, dw, y
    t = torch.randint(0, 3, (140000,), device="cuda")
    small = torch.randn(3, 4096, device="cuda").bfloat16()
    y, dw = _step(t, small, torch.ones(1, 1, dtype=torch.bfloat16, device="cuda").expand(140000, 4, 4096), streams=4)
    assert torch.equal(y[139999, 3], small[t[139999]])
    assert torch.equal(dw[:, 0], (4.0 * torch.bincount(t)).bfloat16())


@gpu
def test_gradients_against_differences():
    """Linear in the table: central differences of sum(g y) err by rounding alone, u / h a term."""
    t, w, g = _inputs(60, 12, 20, torch.float32, 2, seed=3)
    _, dw = _step(t, w, g, scale=1.5, streams=2)
    v = torch.randn_like(w)
    up, down = ((fh.embedding(t, w + h * v, scale=1.5, streams=2).double() * g.double()).sum() for h in (0.25, -0.25))
    want = (dw.double() * v.double()).sum()
    assert abs((up - down) / 0.5 - want) <= 1e-5 * dw.double().norm() * v.double().norm()


@gpu
def test_second_derivatives_go_native():
    t, w, g = _inputs((3, 11), 6, 9, torch.float32, 2)
    g = g.requires_grad_()
    w = w.requires_grad_()
    y = fh.embedding(t, w, scale=2.0, streams=2, padding_idx=4)
    (dw,) = torch.autograd.grad(y, w, g, create_graph=True)
    (got,) = torch.autograd.grad(dw.square().sum(), g)
    keep = (t != 4).float()[..., None, None]
    torch.testing.assert_close(got, (2 * dw.detach() * 2.0)[t].unsqueeze(-2).expand_as(g) * keep)


@gpu
def test_compiled_step_matches():
    f = torch.compile(lambda a, b: fh.embedding(a, b, scale=0.5, streams=3), fullgraph=True, backend="aot_eager")
    for rows, vocab in ((4, 100), (7, 101), (90, 1000)):  # sizes become symbols
        t, w, g = _inputs((rows, 33), 40, vocab, torch.bfloat16, 3)
        leaf = w.clone().requires_grad_()
        y = f(t, leaf)
        (dw,) = torch.autograd.grad(y, leaf, g)
        want = _step(t, w, g, scale=0.5, streams=3)
        assert torch.equal(y, want[0]) and torch.equal(dw, want[1])


@gpu
def test_function_transforms_and_tangents_go_native():
    t, w, _ = _inputs(20, 6, 9, torch.float32)
    torch.testing.assert_close(torch.func.vmap(lambda a: fh.embedding(a, w, scale=2.0))(t), w[t] * 2.0)
    y, dy = torch.func.jvp(lambda b: fh.embedding(t, b, scale=2.0), (w,), (w + 1,))
    torch.testing.assert_close(dy, (w + 1)[t] * 2.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("streams", [None, 3])
def test_cpu_tensors_go_native(dtype, streams):
    t, w, g = _inputs((5, 8), 21, 30, dtype, streams, device="cpu")
    _compare(t, w, g, 1.5, streams, 15)


def test_refusals_on_the_cpu():
    t, w, _ = _inputs(4, 10, 6, torch.float32, device="cpu")
    for args, match in ((dict(streams=0), "streams"), (dict(padding_idx=6), "padding_idx"),
                        (dict(padding_idx=-7), "padding_idx")):
        with pytest.raises(ValueError, match=match):
            fh.embedding(t, w, **args)
    with pytest.raises(ValueError, match="weight"):
        fh.embedding(t, w[0])
    with pytest.raises(IndexError):
        fh.embedding(t + 6, w)
    assert torch.equal(fh.embedding(t, w, padding_idx=-1), w[t])


@gpu
def test_refusals():
    t, w, g = _inputs(4, 10, 6, torch.bfloat16)
    with pytest.raises(RuntimeError):
        fh.embedding(t, w.cpu())
    with pytest.raises(RuntimeError):
        fh.embedding(t.float(), w)
    ops = torch.ops.flash_hypercons
    with pytest.raises(RuntimeError, match="weight"):
        ops._embedding(t, w.cpu(), 1.0, 0, -1)
    with pytest.raises(RuntimeError, match="tokens"):
        ops._embedding(t.float(), w, 1.0, 0, -1)
    with pytest.raises(RuntimeError, match="streams"):
        ops._embedding(t, w, 1.0, -1, -1)
    with pytest.raises(RuntimeError, match="grad"):
        ops._embedding_backward(g[:3], t, 6, 1.0, 0, -1)
    with pytest.raises(RuntimeError, match="grad"):
        ops._embedding_backward(g, t, 0, 1.0, 0, -1)
