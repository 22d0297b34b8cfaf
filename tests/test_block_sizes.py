"""Sizes beyond what the kernels take are composed from native operations, as the entry points say.

Meta tensors stand for tensors of these sizes; nothing is allocated.
"""

import pytest
import torch

import flash_hypercons as fh
from flash_hypercons.ops import block


@pytest.fixture
def eligible(monkeypatch):
    """Meta tensors pass for tensors of a supported device; the operators note their calls."""
    calls = []
    monkeypatch.setattr(block, "_plain", lambda t: True)
    monkeypatch.setattr(block, "_device_supported", lambda index: True)
    monkeypatch.setattr(block, "_NORM", lambda x, *rest: calls.append("norm") or x)
    monkeypatch.setattr(block, "_LINEAR", lambda x, w, *rest: calls.append("linear") or x.new_empty((*x.shape[:-1], len(w))))
    return calls


def _meta(*shape):
    return torch.empty(shape, device="meta", dtype=torch.bfloat16)


@pytest.mark.parametrize("shape,own", [((2**31 - 1, 3), True), ((2**16, 2**15 - 1, 3), True), ((2**31, 1), False),
                                       ((2**16, 2**15, 2), False), ((2, 2**30 - 1), True), ((2, 2**30), False)])
def test_layer_norm(eligible, shape, own):
    y = fh.layer_norm(_meta(*shape))
    assert y.shape == shape and y.dtype == torch.bfloat16 and bool(eligible) == own


@pytest.mark.parametrize("shape,outs,own", [
    ((2**30 - 1, 2), 3, True), ((2**30, 1), 1, False), ((2**15, 2**15, 4), 8, False), ((5, 2**22 - 1), 1, True),
    ((5, 2**22), 1, False), ((5, 8), 2**22 - 1, True), ((5, 8), 2**22, False),
])  # fmt: skip
def test_linear(eligible, shape, outs, own):
    y = fh.linear(_meta(*shape), _meta(outs, shape[-1]))
    assert y.shape == (*shape[:-1], outs) and y.dtype == torch.bfloat16 and bool(eligible) == own
