"""layer_norm, linear and clipping on other streams, from several threads and in captured graphs."""

import threading

import pytest
import torch

import flash_hypercons as fh

pytestmark = pytest.mark.gpu


def _inputs(dtype, m, k, n, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    return normal(m, k), normal(k), normal(k), normal(n, k) * k**-0.5, normal(n), normal(m, n)


def _step(x, scale, shift, w, b, g):
    leaves = [t.detach().requires_grad_() for t in (x, scale, shift, w, b)]
    y = fh.linear(fh.layer_norm(*leaves[:3]), *leaves[3:], activation="silu")
    clipped, norm = fh.clip_grad_norm(torch.autograd.grad(y, leaves, g), 0.5)
    return [y.detach(), *clipped, norm]


# One for each way that a product is taken: few rows, few columns, tiles, slices, FP32.
CASES = [(torch.bfloat16, 3, 512, 4096), (torch.float16, 2000, 4096, 16), (torch.bfloat16, 4000, 520, 4200),
         (torch.bfloat16, 200, 4096, 384), (torch.float32, 300, 1027, 515)]


def test_threads_on_their_own_streams_match_a_single_thread():
    inputs = [_inputs(*case, seed=i) for i, case in enumerate(CASES)]
    want = [_step(*t) for t in inputs]
    torch.cuda.synchronize()
    start, failures = threading.Barrier(len(CASES)), []

    def work(i):
        stream = torch.cuda.Stream()
        start.wait()
        with torch.cuda.stream(stream):
            for _ in range(3):
                got = _step(*inputs[i])
        stream.synchronize()
        if not all(map(torch.equal, got, want[i])):
            failures.append(CASES[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(CASES))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


@pytest.mark.parametrize("case", CASES, ids=str)
def test_graph_replays_match(case):
    """A captured step, replayed on new inputs with eager work between the replays."""
    static = _inputs(*case, seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(*static)
    for seed in range(2, 5):
        for t, new in zip(static, _inputs(*case, seed=seed)):
            t.copy_(new)
        want = _step(*static)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want))
