"""The example's stack of blocks trains, and gives the same tokens one at a time."""

import importlib.util

import pytest
import torch

from tests.conftest import ROOT

spec = importlib.util.spec_from_file_location("hyper_block", ROOT / "examples" / "hyper_block.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


@pytest.mark.parametrize(
    "device,dtype",
    [("cpu", torch.float32), *(pytest.param("cuda", d, marks=pytest.mark.gpu) for d in (torch.float32, torch.bfloat16))],
    ids=str,
)
def test_stack_trains_and_serves(device, dtype):
    torch.manual_seed(1)
    stack = example.Stack(width=40, streams=4, depth=2, device=device, dtype=dtype)
    losses, norms = example.train(stack, steps=25, tokens=64, max_norm=0.5)
    assert all(0 < n < float("inf") for n in norms) and max(norms) > 0.5  # clipped, and not always tiny
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5])
    with torch.no_grad():
        tokens = torch.randn(5, 40).to(device, dtype)
        together, alone = stack(tokens), torch.cat([stack(t.unsqueeze(0)) for t in tokens])
    # Other kernels, other orders of FP32 sums: a few roundings of the storage type at most.
    assert (together - alone).abs().max() <= (1e-4 if dtype == torch.float32 else 0.1) * together.abs().max()


@pytest.mark.gpu
def test_gpu_gradients_match_the_cpu():
    """The same network and data in FP32 on both: gradients agree to FP32 sums' accuracy."""
    grads = []
    for device in ("cpu", "cuda"):
        torch.manual_seed(2)
        stack = example.Stack(width=48, streams=4, depth=2, device=device)
        x = torch.randn(33, 48, generator=torch.Generator().manual_seed(3)).to(device)
        stack(x).square().sum().backward()
        grads.append([p.grad.cpu() for p in stack.parameters()])
    for a, b in zip(*grads):
        assert (a - b).norm() <= 2e-4 * a.norm() + 1e-5
