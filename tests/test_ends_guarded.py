"""The C entry points of embedding and the loss in memory of exactly the size they ask for.

Every array lies in a block of its own whose other bytes, and whose own bytes where it is a result or a
workspace, are 0xFF before the call: NaN in every type, -1 as a place.  So a row that is not written, scratch that
is read before it is written and a byte past an operand that takes part all show as NaN in results, which
are compared with the formulas in 64 bits; and a byte written outside of an array shows in its block.
"""

import ctypes

import pytest
import torch

from tests.test_embedding import _check as _check_embedding
from tests.test_embedding import _formula as _embedding_formula
from tests.test_embedding import _inputs as _embedding_inputs
from tests.test_ends_capi import I64, lib  # noqa: F401
from tests.test_linear_cross_entropy import _check, _formula, _inputs

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
NONE, SUM, MEAN = 0, 1, 2
GUARD = 1 << 16


class Arrays:
    """Arrays with guards around them, `shift` bytes off a multiple of 256."""

    def __init__(self):
        self.blocks = []

    def _block(self, size, shift):
        whole = torch.full((2 * GUARD + size + 512,), 0xFF, dtype=torch.uint8, device="cuda")
        at = GUARD + (-(whole.data_ptr() + GUARD)) % 256 + shift
        self.blocks.append((whole, at, size))
        return whole[at:at + size]

    def copy(self, t, shift=0):
        """An operand: contiguous, with its values."""
        inner = self._block(t.numel() * t.element_size(), shift)
        inner.copy_(t.contiguous().view(-1).view(torch.uint8))
        return inner.view(t.dtype).view(t.shape)

    def empty(self, shape, dtype, shift=0):
        count = 1
        for n in shape:
            count *= n
        size = count * torch.empty((), dtype=dtype).element_size()
        return self._block(size, shift).view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for whole, at, size in self.blocks:
            assert bool((whole[:at] == 0xFF).all()) and bool((whole[at + size:] == 0xFF).all())


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _run(lib, arrays, call, shift=0):  # noqa: F811
    """call(workspace, size), with the size it asks for."""
    size = I64(-1)
    assert call(None, ctypes.byref(size)) == 0, lib.fh_last_error()
    workspace = arrays.empty((size.value,), torch.uint8, shift)
    assert call(workspace.data_ptr() or 16, ctypes.byref(size)) == 0, lib.fh_last_error()


# Tokens searched by each workgroup, sorted in one and in several, by tiles of each size; dense blocks of rows and
# tables that hardly occur.
EMBEDDINGS = [(0, 5, 300, 0), (1, 3, 32768, 0), (700, 450, 5000, 2), (2048, 65, 70001, 0), (1711, 1079, 872, 2),
              (2049, 130, 3000, 3), (4097, 33, 1000, 0), (16385, 9, 262145, 0), (70000, 40, 5000, 0), (140000, 7, 911, 2)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,cols,vocab,streams", EMBEDDINGS)
def test_embedding(lib, tokens, cols, vocab, streams, dtype):  # noqa: F811
    t, w, g = _embedding_inputs(tokens, cols, vocab, dtype, streams, seed=tokens + cols)
    if tokens > 1:
        t[: tokens // 2] = torch.arange(tokens // 2, device="cuda") % vocab
    padding = vocab // 3 if tokens % 2 else None
    want, bound = _embedding_formula(t, w, g, 1.5, streams, padding)
    n = max(1, streams)
    for shift in (0, 16):
        a = Arrays()
        tokens_, w_, g_ = a.copy(t, 8), a.copy(w, shift and 4), a.copy(g, shift and 4)
        y = a.empty((tokens, *((streams,) if streams else ()), cols), dtype, shift and 4)
        dw = a.empty((vocab, cols), dtype, shift and 4)
        assert lib.fh_embedding(tokens_.data_ptr(), w_.data_ptr(), cols, 1.5, n, y.data_ptr(), CODES[dtype], tokens,
                                vocab, cols, _stream()) == 0, lib.fh_last_error()
        _run(lib, a, lambda ws, size: lib.fh_embedding_backward(
            tokens_.data_ptr(), g_.data_ptr(), cols, 1.5, n, -1 if padding is None else padding, dw.data_ptr(), ws, size,
            CODES[dtype], tokens, vocab, cols, _stream()), shift)
        a.check()
        _check_embedding(y, want[0], bound[0], "y")
        _check_embedding(dw, want[1], bound[1], "dw")
        assert torch.equal(g_, g) and torch.equal(w_, w) and torch.equal(tokens_, t)


class Loss:
    """The operands of a loss in guarded arrays, and its calls."""

    def __init__(self, lib, x, w, t, b, reduction, shift):  # noqa: F811
        self.lib, self.a, self.shift = lib, Arrays(), shift
        self.operands = x, w, t, b
        self.x, self.w, self.t = self.a.copy(x, shift), self.a.copy(w, shift), self.a.copy(t, 8)
        self.b = self.a.copy(b, shift and 4) if b is not None else None
        (self.rows, self.cols), self.vocab, self.dtype, self.reduction = x.shape, w.shape[0], x.dtype, reduction
        self.bias_code = CODES[b.dtype if b is not None else x.dtype]
        self.head = (self.x.data_ptr(), self.cols, self.w.data_ptr(), self.cols, self.b.data_ptr() if b is not None else None,
                     self.bias_code, self.t.data_ptr(), -100, reduction)
        self.tail = CODES[x.dtype], self.rows, self.cols, self.vocab, _stream()

    def outputs(self):
        e = lambda shape, dtype: self.a.empty(shape, dtype, self.shift and 4)  # noqa: E731
        return (e((self.rows, self.cols), self.dtype), e((self.vocab, self.cols), self.dtype),
                e((self.vocab,), self.b.dtype) if self.b is not None else None)

    def again(self, g):
        f32, a = torch.float32, self.a
        loss, lse = a.empty((self.rows,) if self.reduction == NONE else (), f32, 4), a.empty((self.rows, 2), f32, 8)
        _run(self.lib, a, lambda ws, size: self.lib.fh_linear_cross_entropy(
            *self.head, loss.data_ptr(), lse.data_ptr(), ws, size, *self.tail), self.shift)
        g_, out = a.copy(g, 4), self.outputs()
        _run(self.lib, a, lambda ws, size: self.lib.fh_linear_cross_entropy_backward(
            *self.head, lse.data_ptr(), g_.data_ptr(), *map(_pointer, out), ws, size, *self.tail), self.shift)
        return self._done(loss, out)

    def ahead(self, g):
        f32, a = torch.float32, self.a
        loss, places = a.empty((), f32, 4), a.empty((1 + self.rows,), torch.int32, 4)
        sums = (a.empty((self.rows, self.cols), f32, self.shift), a.empty((self.vocab, self.cols), f32, self.shift),
                a.empty((self.vocab,), f32, 4) if self.b is not None else None)
        _run(self.lib, a, lambda ws, size: self.lib.fh_linear_cross_entropy_ahead(
            *self.head, loss.data_ptr(), places.data_ptr(), *map(_pointer, sums), ws, size, *self.tail), self.shift)
        g_, out = a.copy(g, 4), self.outputs()
        assert self.lib.fh_linear_cross_entropy_scale(
            g_.data_ptr(), self.t.data_ptr(), -100, self.reduction, places.data_ptr(), *map(_pointer, sums),
            *map(_pointer, out), self.bias_code, *self.tail) == 0, self.lib.fh_last_error()
        return self._done(loss, out)

    def _done(self, loss, out):
        self.a.check()
        for mine, given in zip((self.x, self.w, self.t, self.b), self.operands):
            assert given is None or torch.equal(mine, given)
        return [loss, *out[: 2 + (self.b is not None)]]


def _pointer(t):
    return t.data_ptr() if t is not None else None


# (rows, columns, words, share ignored): one row; two parts and one; many rows of which few have a target, whose sums
# go in more slices; slices of narrow products and of tiles; odd sizes; several chunks of rows and pieces of words.
LOSSES = [(1, 4096, 1000, 0.0), (1, 7, 1, 0.0), (31, 130, 65, 0.2), (128, 72, 4100, 0.1), (129, 72, 4100, 0.1),
          (300, 2056, 300, 0.0), (2000, 136, 777, 0.995), (4096, 264, 2049, 0.9), (1500, 203, 5000, 0.5),
          (520, 16, 31, 0.0), (70000, 8, 33000, 0.4)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,cols,vocab,ignored", LOSSES)
def test_loss(lib, rows, cols, vocab, ignored, dtype):  # noqa: F811
    x, w, t, b = _inputs(rows, cols, vocab, dtype, seed=rows + vocab, ignored=ignored)
    if ignored > 0.9:
        t[1::2] = -100
        t[rows // 2] = vocab - 1  # a target at least
    bias = b if (rows + vocab) % 2 == 0 or rows > 60000 else None
    each, one = torch.rand(rows, device="cuda"), torch.tensor(3.0, device="cuda")
    large = rows > 60000  # its formula takes seconds: once, for both ways at once
    for shift in (0,) if large else (0, 16):
        found = [("ahead", MEAN, one)] + ([] if large and dtype != torch.bfloat16 else [("again", NONE, each)])
        for way, reduction, g in found:
            got = getattr(Loss(lib, x, w, t, bias, reduction, shift), way)(g)
            want, bound = _formula(x, w, t, bias, "none" if reduction == NONE else "mean", g, ahead=way == "ahead")
            for name, a, e, limit in zip(("loss", "dx", "dw", "db"), got, want, bound):
                _check(a, e, limit, f"{way} {name} shift {shift}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [40, 1300])
def test_no_target_in_memory_of_nan(lib, rows, dtype):  # noqa: F811
    """Gradients of no target at all are zeros wherever they are formed."""
    x, w, t, b = _inputs(rows, 136, 777, dtype)
    t[:] = -100
    for way, reduction, g in (("ahead", SUM, torch.tensor(1.0)), ("again", SUM, torch.tensor(1.0)), ("again", NONE, torch.ones(rows))):
        loss, *grads = getattr(Loss(lib, x, w, t, b, reduction, 0), way)(g.cuda())
        assert not loss.any() and not any(d.any() for d in grads)
