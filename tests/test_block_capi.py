"""The C entry points of layer norm, linear and clipping: refusals and workspace sizes, on the CPU.

Nothing here launches a kernel: every call is refused, asks for a size, or has no rows.
"""

import ctypes

import pytest

from tests.test_capi import load

F32, BF16, F16 = 0, 1, 2
P = ctypes.c_void_p
I64 = ctypes.c_int64
A = 0x10000  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    lib = load()
    lib.fh_last_error.restype = ctypes.c_char_p
    lib.fh_layer_norm.argtypes = [P, I64, P, P, ctypes.c_int, ctypes.c_double, P, P, ctypes.c_int, I64, I64, P]
    lib.fh_layer_norm_backward.argtypes = [P, I64, P, I64, P, ctypes.c_int, P, P, P, P, P, P, ctypes.c_int, I64, I64, P]
    lib.fh_linear.argtypes = [P, I64, P, I64, P, ctypes.c_int, P, I64, ctypes.c_int, P, P, P, P, ctypes.c_int, I64, I64,
                              I64, P]
    lib.fh_linear_backward.argtypes = [P, I64, P, I64, P, I64, P, ctypes.c_int, P, P, P, ctypes.c_int, P, P,
                                       ctypes.c_int, I64, I64, I64, P]
    lib.fh_grad_norm.argtypes = [ctypes.c_int, P, P, P, ctypes.c_double, P, P, P, P]
    lib.fh_clip_gradients.argtypes = [ctypes.c_int, P, P, P, P, ctypes.c_double, ctypes.c_double, P, P, P, P]
    return lib


def _norm(lib, x=A, stride=8, param=F32, y=A, dtype=F32, rows=4, cols=8):
    return lib.fh_layer_norm(x, stride, None, None, param, 1e-5, y, None, dtype, rows, cols, None)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(param=BF16), dict(rows=-1), dict(rows=2**31), dict(cols=0),
                                 dict(cols=2**30), dict(x=None), dict(y=None), dict(x=A + 2), dict(stride=-8)],
                         ids=str)
def test_layer_norm_refuses(lib, bad):
    assert _norm(lib, **bad) == 1 and b"layer_norm" in lib.fh_last_error()


def test_no_rows_is_a_no_op(lib):
    assert _norm(lib, x=None, y=None, rows=0) == 0 and lib.fh_last_error() == b""
    size = I64(0)
    assert _linear(lib, ctypes.byref(size), x=None, w=None, y=None, rows=0, workspace=A) == 0


def _norm_backward(lib, workspace, size, dw=A, stats=A, rows=4):
    return lib.fh_layer_norm_backward(A, 8, A, 8, None, F32, stats, A, dw, None, workspace, size, F32, rows, 8, None)


def test_layer_norm_backward_workspace(lib):
    size = I64(-1)
    assert _norm_backward(lib, None, ctypes.byref(size)) == 0 and size.value > 0 and size.value % (2 * 8 * 4) == 0
    assert _norm_backward(lib, None, ctypes.byref(size), dw=None) == 0 and size.value == 0
    assert _norm_backward(lib, None, None) == 1 and b"workspace" in lib.fh_last_error()
    small = I64(4)
    assert _norm_backward(lib, A, ctypes.byref(small)) == 1 and b"bytes" in lib.fh_last_error()
    large = I64(1 << 30)
    assert _norm_backward(lib, A + 4, ctypes.byref(large)) == 1 and b"16-byte aligned" in lib.fh_last_error()
    assert _norm_backward(lib, None, ctypes.byref(size), stats=None) == 1
    assert _norm_backward(lib, None, ctypes.byref(size), rows=0) == 1 and b"no rows" in lib.fh_last_error()


def _linear(lib, size, x=A, w=A, y=A, stride=64, bias=F32, act=0, dtype=F32, rows=4, cols=64, outs=32, workspace=None):
    return lib.fh_linear(x, stride, w, cols, None, bias, None, 0, act, y, None, workspace, size, dtype, rows, cols, outs,
                         None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(bias=F16), dict(rows=-1), dict(cols=0), dict(cols=2**22),
                                 dict(outs=0), dict(outs=2**22), dict(act=5), dict(act=-1), dict(x=None), dict(w=None),
                                 dict(y=None), dict(x=A + 1), dict(stride=-64)], ids=str)
def test_linear_refuses(lib, bad):
    size = I64(0)
    assert _linear(lib, ctypes.byref(size), **bad) == 1 and b"linear" in lib.fh_last_error()


def test_linear_workspace(lib):
    size = I64(-1)
    # 16-bit rows that are no whole vectors are laid out anew; aligned ones of one step are read as they are.
    assert _linear(lib, ctypes.byref(size), dtype=BF16, bias=BF16, cols=64, outs=128, rows=128) == 0 and size.value == 0
    assert _linear(lib, ctypes.byref(size), dtype=BF16, bias=BF16, cols=63, stride=63, outs=128, rows=128) == 0
    assert size.value == 2 * 128 * 64 * 2
    # A long sum with few results goes in slices, whose partial sums are FP32.
    assert _linear(lib, ctypes.byref(size), dtype=F32, cols=4096, stride=4096, rows=64, outs=32) == 0
    assert size.value % (64 * 32 * 4) == 0
    assert _linear(lib, None) == 1 and b"workspace" in lib.fh_last_error()


def test_linear_backward_refuses(lib):
    size = I64(-1)

    def call(saved=None, act=0, dx=A, dw=A, w=A, x=A, rows=4):
        return lib.fh_linear_backward(x, 64, w, 64, A, 32, saved, act, dx, dw, None, F32, None, ctypes.byref(size), F32,
                                      rows, 64, 32, None)

    assert call() == 0
    assert call(act=2) == 1 and b"saved" in lib.fh_last_error()
    assert call(saved=A) == 1 and call(saved=A, act=2) == 0
    assert call(x=None) == 1 and call(x=None, dw=None) == 0
    assert call(w=None) == 1 and call(w=None, dx=None) == 0
    assert call(rows=0) == 1 and b"no rows" in lib.fh_last_error()


def test_clipping_lists(lib):
    size = I64(-1)
    two = (P * 2)(A, A + 4096)
    sizes, dtypes = (I64 * 2)(10, 20), (ctypes.c_int * 2)(F32, BF16)

    def norm(count=2, grads=two, sizes=sizes, dtypes=dtypes, p=2.0, out=A):
        return lib.fh_grad_norm(count, grads, sizes, dtypes, p, out, None, ctypes.byref(size), None)

    assert norm() == 0 and size.value > 0 and size.value % 8 == 0
    assert norm(p=float("inf")) == 0 and norm(p=1.0) == 0
    assert norm(p=3.0) == 1 and b"norm_type" in lib.fh_last_error()
    assert norm(count=-1) == 1 and norm(grads=None) == 1 and norm(out=None) == 1
    assert norm(sizes=(I64 * 2)(10, -1)) == 1 and norm(dtypes=(ctypes.c_int * 2)(F32, 9)) == 1
    assert norm(grads=(P * 2)(A, None)) == 1 and norm(grads=(P * 2)(A, A + 1)) == 1
    assert norm(grads=(P * 2)(A, None), sizes=(I64 * 2)(10, 0)) == 0  # an empty array may be null
    assert norm(count=0, grads=None, sizes=None, dtypes=None) == 0 and size.value == 0

    def clip(out):
        return lib.fh_clip_gradients(2, two, out, sizes, dtypes, 2.0, 1.0, A, None, ctypes.byref(size), None)

    assert clip(None) == 0 and clip((P * 2)(A, A)) == 0
    assert clip((P * 2)(A, None)) == 1 and b"clip_gradients" in lib.fh_last_error()
