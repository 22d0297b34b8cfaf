"""The global gradient norm and clipping, against 64 bits.

The norm's sums are FP64 and its result one FP32 rounding (bound 2^-23); the scaling rounds the
factor and the product to FP32 (2^-23) and once to the storage type.
"""

import math

import pytest
import torch

import flash_hypercons as fh
from tests.mixcheck import floor, half_ulp

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TYPES = [1.0, 2.0, math.inf]
gpu = pytest.mark.gpu


def _norm(tensors, p):
    flat = torch.cat([t.detach().double().cpu().reshape(-1) for t in tensors])
    return torch.linalg.vector_norm(flat, p)


def _check(tensors, max_norm, p=2.0, inplace_too=True):
    before = [t.clone() for t in tensors]
    want = _norm(tensors, p)
    factor = min(1.0, float(max_norm / (want + 1e-6)))
    got = fh.grad_norm(tensors, p)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(got.double().cpu() - want) <= 2.0**-23 * want
    clipped, norm = fh.clip_grad_norm(tensors, max_norm, p)
    assert torch.equal(norm, got)
    for t, b, c in zip(tensors, before, clipped):
        assert torch.equal(t, b) and c.dtype == t.dtype and c.shape == t.shape
        exact = t.double().cpu() * factor
        limit = (half_ulp(t.dtype) + 2.0**-22) * exact.abs() + floor(t.dtype)
        assert bool(((c.double().cpu() - exact).abs() <= limit).all())
    if inplace_too:
        params = []
        for t in tensors:
            q = torch.nn.Parameter(torch.zeros_like(t))
            q.grad = t
            params.append(q)
        versions = [t._version for t in tensors]
        assert torch.equal(fh.clip_grad_norm_(params, max_norm, p), got)
        for t, c, b, v in zip(tensors, clipped, before, versions):
            assert torch.equal(t, c) and t._version > v
            if factor == 1.0:
                assert torch.equal(t, b)


def _tensors(sizes, dtypes, device="cuda", seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn(s, generator=gen, device=device) * 10.0 ** -(i % 3)).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(sizes)]


SIZES = [(1,), (2,), (7,), (8, 9), (255,), (4097,), (31, 33), (3, 5, 7), (16385,), (8192,), (16384,), (64, 513)]


@gpu
@pytest.mark.parametrize("p", TYPES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_sizes_and_norms(dtype, p):
    for share in (0.25, 4.0):
        tensors = _tensors(SIZES, [dtype])
        _check(tensors, share * float(_norm(tensors, p)), p)


@gpu
def test_mixed_types():
    tensors = _tensors(SIZES, DTYPES)
    _check(tensors, 0.5)


@gpu
@pytest.mark.parametrize("count", [1, 95, 96, 97, 300])
def test_many_tensors(count):
    _check(_tensors([(1 + (37 * i) % 501,) for i in range(count)], DTYPES, seed=count), 1.0)


@gpu
def test_one_large_tensor():
    _check(_tensors([(5_000_011,)], [torch.bfloat16]), 10.0)


@gpu
def test_empty_tensors():
    _check(_tensors([(0,), (5,), (3, 0), (9,)], [torch.float32]), 0.1)
    empty = [torch.zeros(0, device="cuda")]
    assert fh.grad_norm(empty).item() == 0.0
    clipped, norm = fh.clip_grad_norm(empty, 1.0)
    assert norm.item() == 0.0 and clipped[0].numel() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views(dtype):
    base = _tensors([(12, 40)], [dtype])[0]
    _check([base.t(), base.clone().reshape(3, 4, 40).permute(2, 0, 1)], 1.0)  # dense in another order
    wide = _tensors([(12, 90)], [dtype], seed=1)[0]
    edge = wide.clone()
    _check([wide[:, 1:40], wide[:, 40:81:2]], 1.0)  # with gaps: through copies, and interleaved
    assert torch.equal(wide[:, :1], edge[:, :1]) and torch.equal(wide[:, 41:81:2], edge[:, 41:81:2])
    flat = _tensors([(501,)], [dtype], seed=2)[0]
    _check([flat[1:130], flat[131:500]], 1.0)  # at odd elements, side by side
    _check([flat[:1].expand(77)], 1.0, inplace_too=False)


@gpu
def test_values_whose_squares_leave_float32():
    for scale in (1e25, 1e-30):
        tensors = [t * scale for t in _tensors([(1000,), (37,)], [torch.float32])]
        _check(tensors, 1.0)


@gpu
@pytest.mark.parametrize("p", TYPES)
def test_infinity_and_nan(p):
    tensors = _tensors([(3000,), (50,)], [torch.float32])
    tensors[0][2999] = float("inf")
    clipped, norm = fh.clip_grad_norm(tensors, 1.0, p)
    assert norm.item() == math.inf
    assert clipped[0][2999].isnan() and not clipped[0][:2999].any() and not clipped[1].any()
    tensors[1][3] = float("nan")
    clipped, norm = fh.clip_grad_norm(tensors, 1.0, p)
    assert norm.isnan() and all(c.isnan().all() for c in clipped)


@gpu
def test_results_are_the_same_bits_again():
    tensors = _tensors([(100_003,), (77, 1025), (9,)], DTYPES)
    first, again = fh.clip_grad_norm(tensors, 0.3), fh.clip_grad_norm(tensors, 0.3)
    assert torch.equal(first[1], again[1]) and all(map(torch.equal, first[0], again[0]))


@gpu
def test_graph_replays_match():
    """A captured clipping, replayed on new gradients with eager work between the replays."""
    tensors = _tensors(SIZES, DTYPES)
    for _ in range(2):
        fh.clip_grad_norm(tensors, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clipped, norm = fh.clip_grad_norm(tensors, 0.5)
    for seed in range(3):
        for t, new in zip(tensors, _tensors(SIZES, DTYPES, seed=10 + seed)):
            t.copy_(new)
        want, want_norm = fh.clip_grad_norm(tensors, 0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want_norm) and all(map(torch.equal, clipped, want))


@gpu
def test_other_norms_and_missing_gradients_go_native():
    tensors = _tensors([(40,), (9, 9)], [torch.float32])
    assert abs(fh.grad_norm(tensors, 3.0).item() - _norm(tensors, 3.0).item()) < 1e-5
    params = [torch.nn.Parameter(t) for t in tensors]
    params[0].grad = tensors[0].clone()
    assert abs(fh.clip_grad_norm_(params, 1e9).item() - _norm(tensors[:1], 2.0).item()) < 1e-5
    assert params[1].grad is None


@pytest.mark.parametrize("p", TYPES + [3.0])
@pytest.mark.parametrize("dtype", DTYPES + [torch.float64], ids=str)
def test_cpu_tensors_go_native(dtype, p):
    tensors = _tensors([(40,), (0,), (9, 9)], [dtype], device="cpu")
    want = _norm(tensors, p)
    assert abs(fh.grad_norm(tensors, p).double() - want) <= 2.0**-22 * want
    clipped, norm = fh.clip_grad_norm(tensors, 0.25, p)
    assert abs(_norm(clipped, p) - 0.25) <= (half_ulp(dtype) if dtype != torch.float64 else 0) + 1e-5
    params = [torch.nn.Parameter(torch.zeros_like(t)) for t in tensors]
    for q, t in zip(params, tensors):
        q.grad = t.clone()
    assert torch.equal(fh.clip_grad_norm_(params, 0.25, p), norm)
    assert all(torch.equal(q.grad, c) for q, c in zip(params, clipped))


def test_nothing_to_clip():
    assert fh.grad_norm([]).item() == 0.0
    assert fh.clip_grad_norm([], 1.0)[0] == []
    assert fh.clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0).item() == 0.0
    one = torch.nn.Parameter(torch.ones(4))
    one.grad = torch.full((4,), 2.0)
    assert fh.clip_grad_norm_(one, 1.0).item() == 4.0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_nonfinite_norms_raise_where_asked(device):
    p = torch.nn.Parameter(torch.zeros(5, device=device))
    p.grad = torch.full((5,), float("inf"), device=device)
    with pytest.raises(RuntimeError, match="global norm"):
        fh.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert p.grad.isinf().all()


@gpu
def test_refusals():
    t = torch.ones(30, device="cuda")

    def clip(*grads):
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for q, g in zip(params, grads):
            q.grad = g
        return fh.clip_grad_norm_(params, 1.0)

    with pytest.raises(RuntimeError, match="share memory"):
        clip(t, t)
    with pytest.raises(RuntimeError, match="share memory"):
        clip(t[:20], t[10:])
    with pytest.raises(RuntimeError, match="share memory"):
        clip(t[:1].expand(5))
    assert torch.equal(t, torch.ones_like(t))
    with pytest.raises(RuntimeError, match="norm_type"):
        torch.ops.flash_hypercons._grad_norm([t], 3.0)
