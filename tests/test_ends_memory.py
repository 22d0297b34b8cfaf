"""What the loss asks for: workspaces that do not grow with the batch beyond its own rows."""

import ctypes

import pytest

from tests.test_ends_capi import BF16, F16, F32, I64, _ahead, _backward, lib  # noqa: F401

MIB = 1 << 20


def _size(call, lib, **args):  # noqa: F811
    size = I64(-1)
    assert call(lib, ctypes.byref(size), **args) == 0, lib.fh_last_error()
    return size.value


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", [(4096, 32768), (1 << 20, 131072), (1 << 22, 32768), ((1 << 24) - 1, 1000)])
def test_a_bias_takes_sums_of_one_chunk(lib, dtype, rows, vocab):  # noqa: F811
    """Column sums of dz: a 64th of a chunk's 2 GiB of dz, as FP32, whatever the number of chunks."""
    args = dict(dtype=dtype, bias_dtype=dtype, rows=rows, cols=64, vocab=vocab)
    for call in (_ahead, _backward):
        more = _size(call, lib, **args) - _size(call, lib, **args, db=None)
        assert 0 <= more <= 65 * MIB, call.__name__


@pytest.mark.parametrize("call", [_ahead, _backward])
@pytest.mark.parametrize("rows,vocab", [(1 << 16, 131072), (1 << 20, 131072), (1 << 22, 32768), ((1 << 24) - 1, 4096)])
def test_a_batch_takes_its_rows_and_one_chunk(lib, call, rows, vocab):  # noqa: F811
    """2 GiB of dz, what goes with it, and for each row its gathered columns and a few numbers."""
    cols = 64
    size = _size(call, lib, dtype=BF16, bias_dtype=BF16, rows=rows, cols=cols, vocab=vocab)
    own = rows * (cols * 2 + 64)  # x's rows, where they are, targets, losses, factors
    dx = rows * cols * 4 if call is _backward else 0  # the sum over pieces of the vocabulary
    assert size <= (1 << 31) + 512 * MIB + own + dx
