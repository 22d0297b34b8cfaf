"""Embedding, blocks and loss in one network: the example of a word model, trained and scored."""

import importlib.util

import pytest
import torch

import flash_hypercons as fh
from tests.conftest import ROOT

spec = importlib.util.spec_from_file_location("word_model", ROOT / "examples" / "word_model.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)
gpu = pytest.mark.gpu


@pytest.mark.parametrize(
    "device,dtype",
    [("cpu", torch.float32), *(pytest.param("cuda", d, marks=gpu) for d in (torch.float32, torch.bfloat16))],
    ids=str,
)
def test_model_runs(device, dtype):
    """Trains, scores positions together and by themselves.  How far the loss falls is not looked at."""
    torch.manual_seed(1)
    model = example.WordModel(words=97, width=40, depth=1, device=device, dtype=dtype)
    losses, norms = example.train(model, steps=3, count=40, length=30)
    assert all(0 < v < float("inf") for v in losses + norms)
    with torch.no_grad():
        tokens, targets = (t.to(device) for t in example.sequences(97, 3, 10, torch.Generator().manual_seed(2)))
        together = model(tokens, targets, "none")
        alone = torch.cat([model(t.view(1), n.view(1), "none") for t, n in zip(tokens, targets)])
    assert not together[targets == example.PADDING].any()
    # Other kernels, other orders of FP32 sums: a few roundings of the storage type at most.
    assert (together - alone).abs().max() <= (1e-4 if dtype == torch.float32 else 0.1) * (1 + together.abs().max())


@gpu
@pytest.mark.parametrize("count", [3, 50])  # logits formed again, and gradients with the loss
def test_gradients_match_the_cpu(count):
    """The same network and data in FP32 on both; the table's gradient adds those of both ends."""
    grads = []
    for device in ("cpu", "cuda"):
        torch.manual_seed(2)
        model = example.WordModel(words=301, width=48, device=device)
        tokens, targets = example.sequences(301, count, 20, torch.Generator().manual_seed(3))
        model(tokens.to(device), targets.to(device)).backward()
        grads.append([p.grad.cpu() for p in model.parameters()])
    assert grads[0][0].any()
    for a, b in zip(*grads):
        assert (a - b).norm() <= 2e-4 * a.norm() + 1e-6


@gpu
@pytest.mark.parametrize("count", [2, 60])
def test_gradients_against_differences(count):
    """Central differences of the loss along the gradient, h = 2^-9 of a unit step: FP32 rounding of the loss,
    2^-20 or so, over 2 h |g| stays below 1% for |g| above 0.03, and the third derivative below that."""
    torch.manual_seed(4)
    model = example.WordModel(words=200, width=32, depth=1, device="cuda")
    tokens, targets = (t.cuda() for t in example.sequences(200, count, 20, torch.Generator().manual_seed(5)))
    model(tokens, targets).backward()
    norm = fh.grad_norm([p.grad for p in model.parameters()]).item()
    assert norm > 0.03
    value = []
    for sign in (1, -1):
        with torch.no_grad():
            moved = [p + sign * 2.0**-9 * p.grad / norm for p in model.parameters()]
            value.append(torch.func.functional_call(
                model, dict(zip((n for n, _ in model.named_parameters()), moved)), (tokens, targets, "none")).double().sum()
                / (targets != example.PADDING).sum())
    assert abs((value[0] - value[1]) / 2.0**-8 - norm) <= 2e-2 * norm
