"""The C entry points of embedding and the loss: refusals and workspace sizes, on the CPU.

Nothing here launches a kernel: every call is refused, asks for a size, or has no tokens.
"""

import ctypes

import pytest

from tests.test_capi import load

F32, BF16, F16 = 0, 1, 2
NONE, SUM, MEAN = 0, 1, 2
P = ctypes.c_void_p
I64 = ctypes.c_int64
INT = ctypes.c_int
A = 0x10000  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    lib = load()
    lib.fh_last_error.restype = ctypes.c_char_p
    lib.fh_embedding.argtypes = [P, P, I64, ctypes.c_double, INT, P, INT, I64, I64, I64, P]
    lib.fh_embedding_backward.argtypes = [P, P, I64, ctypes.c_double, INT, I64, P, P, P, INT, I64, I64, I64, P]
    head = [P, I64, P, I64, P, INT, P, I64, INT]
    lib.fh_linear_cross_entropy.argtypes = head + [P, P, P, P, INT, I64, I64, I64, P]
    lib.fh_linear_cross_entropy_backward.argtypes = head + [P, P, P, P, P, P, P, INT, I64, I64, I64, P]
    lib.fh_linear_cross_entropy_ahead.argtypes = head + [P, P, P, P, P, P, P, INT, I64, I64, I64, P]
    lib.fh_linear_cross_entropy_scale.argtypes = [P, P, I64, INT, P, P, P, P, P, P, P, INT, INT, I64, I64, I64, P]
    return lib


def _embedding(lib, tokens=A, weight=A, stride=8, streams=1, y=A, dtype=F32, count=4, vocab=5, cols=8):
    return lib.fh_embedding(tokens, weight, stride, 1.0, streams, y, dtype, count, vocab, cols, None)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(count=-1), dict(count=2**28), dict(vocab=0), dict(vocab=2**28),
                                 dict(cols=0), dict(cols=2**24), dict(streams=0), dict(streams=2**16),
                                 dict(tokens=None), dict(tokens=A + 4), dict(weight=None), dict(weight=A + 2),
                                 dict(y=None), dict(stride=-8)], ids=str)
def test_embedding_refuses(lib, bad):
    assert _embedding(lib, **bad) == 1 and b"embedding" in lib.fh_last_error()


def test_no_tokens_is_a_no_op(lib):
    assert _embedding(lib, tokens=None, weight=None, y=None, count=0) == 0 and lib.fh_last_error() == b""


def _embedding_backward(lib, workspace, size, grad=A, dw=A, dtype=F32, count=4, vocab=5, cols=8):
    return lib.fh_embedding_backward(A, grad, 8, 1.0, 1, -1, dw, workspace, size, dtype, count, vocab, cols, None)


def test_embedding_backward_workspace(lib):
    size = I64(-1)
    assert _embedding_backward(lib, None, ctypes.byref(size)) == 0 and size.value == 0  # few tokens need none
    assert _embedding_backward(lib, None, ctypes.byref(size), count=5000, vocab=100) == 0
    assert size.value >= 5000 * 16 + 5000 // 64 * 2 * 8 * 4  # two pairs of keys and places, and partial sums
    small = I64(64)
    assert _embedding_backward(lib, A, ctypes.byref(small), count=5000) == 1 and b"bytes" in lib.fh_last_error()
    assert _embedding_backward(lib, None, None) == 1 and b"workspace" in lib.fh_last_error()
    assert _embedding_backward(lib, None, ctypes.byref(size), dw=None) == 1
    assert _embedding_backward(lib, None, ctypes.byref(size), grad=A + 1) == 1
    assert _embedding_backward(lib, None, ctypes.byref(size), grad=None, count=0) == 0


def _head(x=A, stride=64, w=A, bias=None, bias_dtype=F32, targets=A, reduction=MEAN):
    return x, stride, w, 64, bias, bias_dtype, targets, -100, reduction


def _loss(lib, size, loss=A, lse=A, workspace=None, dtype=F32, rows=4, cols=64, vocab=32, **head):
    return lib.fh_linear_cross_entropy(*_head(**head), loss, lse, workspace, size, dtype, rows, cols, vocab, None)


BAD = [dict(dtype=3), dict(bias_dtype=F16), dict(rows=-1), dict(rows=2**24), dict(cols=0), dict(cols=2**22),
       dict(vocab=0), dict(vocab=2**22), dict(reduction=-1), dict(reduction=3), dict(x=None), dict(w=None),
       dict(targets=None), dict(targets=A + 4), dict(x=A + 1), dict(stride=-64), dict(bias=A + 2), dict(rows=0),
       dict(loss=None), dict(loss=A + 2)]


@pytest.mark.parametrize("bad", BAD + [dict(lse=None), dict(lse=A + 2)], ids=str)
def test_loss_refuses(lib, bad):
    size = I64(0)
    assert _loss(lib, ctypes.byref(size), **bad) == 1 and b"linear_cross_entropy" in lib.fh_last_error()


def _ahead(lib, size, loss=A, places=A, dx=A, dw=A, db=A, workspace=None, dtype=F32, rows=4, cols=64, vocab=32, **head):
    return lib.fh_linear_cross_entropy_ahead(*_head(**head), loss, places, dx, dw, db, workspace, size, dtype, rows, cols,
                                             vocab, None)


@pytest.mark.parametrize("bad", BAD + [dict(reduction=NONE), dict(places=None), dict(places=A + 2), dict(dx=A + 1),
                                       dict(dw=A + 2), dict(db=A + 2)], ids=str)
def test_loss_ahead_refuses(lib, bad):
    size = I64(0)
    assert _ahead(lib, ctypes.byref(size), **bad) == 1 and b"linear_cross_entropy" in lib.fh_last_error()


def test_loss_workspaces(lib):
    size = I64(-1)
    assert _loss(lib, ctypes.byref(size), dtype=BF16, bias_dtype=BF16, rows=512, cols=64, vocab=4096) == 0
    # The gathered rows, and a maximum and a sum for each 64 logits of a row; not the logits.
    assert 512 * 64 * 2 + 512 * 64 * 8 <= size.value < 512 * 4096 * 2
    assert _loss(lib, None) == 1 and b"workspace" in lib.fh_last_error()
    small = I64(16)
    assert _loss(lib, ctypes.byref(small), workspace=A) == 1 and b"bytes" in lib.fh_last_error()
    # At most 2 GiB of a vocabulary's or a batch's gradients at a time.
    for call in (_ahead, _backward):
        assert call(lib, ctypes.byref(size), dtype=BF16, bias_dtype=BF16, rows=65536, cols=64, vocab=131072) == 0
        assert 2**31 <= size.value < 2**31 + 2**30
    assert _ahead(lib, ctypes.byref(size), dx=None, dw=None, db=None) == 0


def _backward(lib, size, lse=A, grad=A, dx=A, dw=A, db=A, dtype=F32, rows=4, cols=64, vocab=32, **head):
    return lib.fh_linear_cross_entropy_backward(*_head(**head), lse, grad, dx, dw, db, None, size, dtype, rows, cols,
                                                vocab, None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(rows=0), dict(lse=None), dict(grad=None), dict(grad=A + 2),
                                 dict(dx=A + 2), dict(dw=A + 1), dict(db=A + 2), dict(x=None)], ids=str)
def test_loss_backward_refuses(lib, bad):
    size = I64(0)
    assert _backward(lib, ctypes.byref(size), **bad) == 1 and b"linear_cross_entropy" in lib.fh_last_error()
    assert _backward(lib, ctypes.byref(size), dx=None, dw=None, db=None) == 0


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(rows=0), dict(reduction=NONE), dict(grad=None), dict(places=None),
                                 dict(dx_sums=None), dict(dw_sums=A + 2), dict(db_sums=None), dict(dx=A + 2)], ids=str)
def test_loss_scale_refuses(lib, bad):
    a = dict(grad=A, targets=A, reduction=MEAN, places=A, dx_sums=A, dw_sums=A, db_sums=A, dx=A, dw=A, db=A, dtype=F32,
             rows=4)
    a.update(bad)
    rc = lib.fh_linear_cross_entropy_scale(a["grad"], a["targets"], -100, a["reduction"], a["places"], a["dx_sums"],
                                           a["dw_sums"], a["db_sums"], a["dx"], a["dw"], a["db"], F32, a["dtype"],
                                           a["rows"], 64, 32, None)
    assert rc == 1 and b"linear_cross_entropy" in lib.fh_last_error()
