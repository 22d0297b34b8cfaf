"""embedding and linear_cross_entropy on other streams, from several threads and in captured graphs."""

import threading

import pytest
import torch

import flash_hypercons as fh

pytestmark = pytest.mark.gpu


def _inputs(dtype, tokens, cols, vocab, reduction, seed, share=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    t = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    n = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    n[torch.rand(tokens, generator=gen, device="cuda") < share] = -100
    return (t, n, (normal(vocab, cols) * cols**-0.5).to(dtype), normal(vocab).to(dtype),
            normal(tokens).abs() if reduction == "none" else normal().abs())


def _step(reduction, t, n, table, bias, g):
    leaves = [a.detach().requires_grad_() for a in (table, bias)]
    streams = fh.embedding(t, leaves[0], scale=2.0, streams=2, padding_idx=0)
    loss = fh.linear_cross_entropy(streams[:, 1] + streams[:, 0], leaves[0], n, leaves[1], reduction=reduction)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, g)]


# One for each way: few tokens and many, rows by themselves and together, logits again and gradients ahead, FP32.
CASES = [(torch.bfloat16, 3, 512, 4096, "none"), (torch.float16, 700, 256, 3000, "mean"),
         (torch.bfloat16, 2500, 264, 5000, "mean"), (torch.float16, 6000, 64, 2001, "sum"),
         (torch.float32, 300, 203, 1027, "mean")]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_threads_on_their_own_streams_match_a_single_thread():
    inputs = [_inputs(*case, seed=i) for i, case in enumerate(CASES)]
    want = [_step(case[4], *t) for case, t in zip(CASES, inputs)]
    torch.cuda.synchronize()
    start, failures = threading.Barrier(len(CASES)), []

    def work(i):
        stream = torch.cuda.Stream()
        start.wait()
        with torch.cuda.stream(stream):
            for _ in range(3):
                got = _step(CASES[i][4], *inputs[i])
        stream.synchronize()
        if not _same(got, want[i]):
            failures.append(CASES[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(CASES))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def _capture(case, static, pool=None):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(case[4], *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool):
        got = _step(case[4], *static)
    return graph, got


@pytest.mark.parametrize("case", CASES, ids=str)
def test_graph_replays_match(case):
    """A captured step, replayed on new inputs, whose share of targets changes, with eager work between."""
    static = _inputs(*case, seed=1)
    graph, got = _capture(case, static)
    for seed, share in ((2, 0.0), (3, 0.9), (4, 1.0), (5, 0.3)):
        for t, new in zip(static, _inputs(*case, seed=seed, share=share)):
            t.copy_(new)
        want = _step(case[4], *static)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(got, want):
            torch.testing.assert_close(a, e, rtol=0, atol=0, equal_nan=True)


def test_two_graphs_of_one_pool():
    """Graphs that share their memory, replayed in turn: nothing of a call stays in its workspace."""
    statics = [_inputs(*case, seed=i) for i, case in enumerate(CASES[1:3])]
    first = _capture(CASES[1], statics[0])
    want = [t.clone() for t in _step("mean", *statics[0])]
    second = _capture(CASES[2], statics[1], pool=first[0].pool())
    for _ in range(3):
        first[0].replay()
        torch.cuda.synchronize()
        assert _same(first[1], want)
        second[0].replay()
        torch.cuda.synchronize()
        assert _same(second[1], _step("mean", *statics[1]))


def test_operands_of_another_stream():
    """Work queued on one stream, whose results another one uses after waiting for it."""
    inputs = _inputs(*CASES[2], seed=7)
    want = _step("mean", *inputs)
    stream = torch.cuda.Stream()
    moved = [t.clone() for t in inputs]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _step("mean", *moved)
    torch.cuda.current_stream().wait_stream(stream)
    assert _same(got, want)
