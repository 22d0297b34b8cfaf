"""Workloads of the block between two stream mixings, as programs run them, for timing and for checking results.

Three operators: ``layer_norm`` (rows normalised, scaled and shifted), ``linear`` (a matrix product with
bias, activation and residual added in its epilogue) and the global gradient norm with clipping
(``clip_grad_norm`` into new tensors, ``clip_grad_norm_`` in place).  The first two run forward alone
(inference) or forward + gradients (training).

A case is a dict:

* ``op``: "norm", "linear" or "clip"; ``dtype``;
* norm: ``tokens``, ``cols``, ``streams`` (above 1 the rows are the first stream of ``[tokens, streams, cols]``
  storage, read in place), ``step`` (gradients as well);
* linear: ``tokens``, ``cols`` (of x), ``outs`` (rows of the weight), ``act``, ``residual``, ``step``;
* clip: ``layers`` of six tensors each (norm weight and bias, two products' weights and biases) of widths
  ``cols`` and ``outs``, ``factor`` (the norm over the allowed one), ``inplace``.
"""

import math
import sys
from pathlib import Path

import torch

own = False  # True: the package's operators; False: plain torch operations in FP32

_ROOT = Path(__file__).resolve().parents[1]
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5


def _package():
    path = str(_ROOT / "flash-hyperconnections_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_hypercons

    return flash_hypercons


def _norm(name, dtype, tokens, cols, streams=1, step=True):
    return {"name": name, "op": "norm", "dtype": dtype, "tokens": tokens, "cols": cols, "streams": streams,
            "step": step}


def _linear(name, dtype, tokens, cols, outs, act="none", residual=False, step=True):
    return {"name": name, "op": "linear", "dtype": dtype, "tokens": tokens, "cols": cols, "outs": outs, "act": act,
            "residual": residual, "step": step}


def _clip(name, dtype, layers, cols, outs, factor, inplace=False):
    return {"name": name, "op": "clip", "dtype": dtype, "layers": layers, "cols": cols, "outs": outs,
            "factor": factor, "inplace": inplace}


def listed():
    return [
        # Serving: one decode step of 64 sequences, the block's input being one of four streams.
        _norm("norm_bf16_t64_c4096", "bf16", 64, 4096, streams=4, step=False),
        # Training: a long batch.
        _norm("norm_bf16_t16384_c4096_step", "bf16", 16384, 4096),
        # Training: four streams normalised together, the input of the mixing generator.
        _norm("norm_f16_t2048_c16384_step", "f16", 2048, 16384),
        # Single precision, a width that is no whole number of vectors.
        _norm("norm_f32_t1500_c1027_step", "f32", 1500, 1027),
        # Serving: a single token through the wide product of a feed-forward block.
        _linear("linear_bf16_t1_k4096_n16384_gelu", "bf16", 1, 4096, 16384, "gelu", step=False),
        # Serving: 64 sequences through the narrow product, added to the stream that the block read.
        _linear("linear_bf16_t64_k16384_n4096_res", "bf16", 64, 16384, 4096, residual=True, step=False),
        # Training: a long batch through the wide product; the largest.
        _linear("linear_bf16_t16384_k4096_n16384_gelu_step", "bf16", 16384, 4096, 16384, "gelu"),
        # Training: the generator of a 4 x 4 mixing matrix from each token's four streams.
        _linear("linear_bf16_t16384_k16384_n16_step", "bf16", 16384, 16384, 16),
        # Single precision, odd sizes, activation and residual together.
        _linear("linear_f32_t1500_k1027_n771_silu_res_step", "f32", 1500, 1027, 771, "silu", True),
        # A unit test or a small model: call latency.
        _clip("clip_f32_l2_c64", "f32", 2, 64, 256, 8.0),
        # Training: all gradients of ten feed-forward blocks, over the allowed norm.
        _clip("clip_bf16_l10_c2048", "bf16", 10, 2048, 8192, 3.0),
        # An ordinary step, whose norm is allowed: the gradients stay as they are.  Odd sizes.
        _clip("clip_f32_l6_c1027_inplace", "f32", 6, 1027, 4093, 0.5, True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width over the logarithm of the range: whole vectors mostly, as models have, odd ones too."""
    w = _log_int(rng, low, high)
    return w if rng.random() < 0.35 or w < 64 else w - w % 64


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "clip"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if op == "norm":
        cols, streams = _width(rng, 33, 16384), rng.choice((1, 1, 2, 4))
        tokens = _log_int(rng, 1, min(16384, (1 << 27) // (cols * streams)))
        case = _norm("", dtype, tokens, cols, streams, rng.random() < 0.6)
    elif op == "linear":
        cols, outs = _width(rng, 33, 16384), _width(rng, 9, 16384)
        most = 1 << (36 if dtype == "f32" else 38)
        tokens = _log_int(rng, 1, max(1, min(16384, most // (cols * outs))))
        act = rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu"))
        case = _linear("", dtype, tokens, cols, outs, act, rng.random() < 0.4, rng.random() < 0.6)
    else:
        cols = _width(rng, 33, 2048)
        outs = _width(rng, cols, 4 * cols)
        case = _clip("", dtype, rng.randint(1, 10), cols, outs, rng.choice((0.5, 1.5, 8.0)))
        case["inplace"] = case["factor"] < 1
    del case["name"]
    return case


def _shapes(case):
    c, o = case["cols"], case["outs"]
    return [(c,), (c,), (o, c), (o,), (c, o), (c,)] * case["layers"]


def _inputs(case, seed):
    """The tensors of a case in its dtype, by name; "g" is the upstream gradient of a step."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale)

    if case["op"] == "clip":
        # Gradients of layers differ in size by orders of magnitude.
        return {"grads": [normal(*s, scale=10.0 ** -(1 + i % 4)).to(dtype) for i, s in enumerate(_shapes(case))]}
    t, c = case["tokens"], case["cols"]
    if case["op"] == "norm":
        # Residual streams: each token of its own size, off zero, a few features much larger.
        x = normal(t, case["streams"], c).mul_(normal(t, 1, 1, scale=0.5).exp_()).add_(0.3)
        x[..., :: 97] *= 8.0
        got = {"x": x.to(dtype)[:, 0], "weight": normal(c, scale=0.2).add_(1.0).to(dtype),
               "bias": normal(c, scale=0.1).to(dtype)}
        if case["step"]:
            got["g"] = normal(t, c).to(dtype)
        return got
    o = case["outs"]
    got = {"x": normal(t, c).to(dtype), "weight": normal(o, c, scale=c**-0.5).to(dtype),
           "bias": normal(o, scale=0.1).to(dtype)}
    if case["residual"]:
        got["residual"] = normal(t, o).to(dtype)
    if case["step"]:
        got["g"] = normal(t, o).to(dtype)
    return got


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["op"] == "clip":
        norm = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt().item()
        state["max_norm"] = norm / case["factor"]
        if case["inplace"]:
            # What a program has: parameters that hold their gradients.
            state["params"] = [torch.nn.Parameter(torch.zeros_like(g)) for g in state["grads"]]
            list(map(lambda p, g: setattr(p, "grad", g), state["params"], state["grads"]))
    elif case["step"]:
        state["args"] = [state[k].requires_grad_() for k in ("x", "weight", "bias", "residual") if k in state]
    return state


# ---- the package's operators ------------------------------------------------------------------


def _run_own(s):
    fh, case = _package(), s["case"]
    if case["op"] == "clip":
        if case["inplace"]:
            norm = fh.clip_grad_norm_(s["params"], s["max_norm"])
            return [norm, *[p.grad for p in s["params"]]]
        clipped, norm = fh.clip_grad_norm(s["grads"], s["max_norm"])
        return [norm, *clipped]
    if case["op"] == "norm":
        y = fh.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
    else:
        act = None if case["act"] == "none" else case["act"]
        y = fh.linear(s["x"], s["weight"], s["bias"], activation=act, residual=s.get("residual"))
    return [y, *torch.autograd.grad(y, s["args"], s["g"])] if case["step"] else [y]


# ---- plain forms -------------------------------------------------------------------------------


def _plain_clip(s):
    grads = s["grads"]
    norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    clipped = [(g.float() * scale).to(g.dtype) for g in grads]
    return [norm, *([g.copy_(c) for g, c in zip(grads, clipped)] if s["case"]["inplace"] else clipped)]


def _plain_norm(s):
    dtype = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    d = x - x.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    n = d * r
    out = [n * w + b]
    if s["case"]["step"]:
        g = s["g"].float()
        gw = g * w
        dx = (gw - gw.mean(-1, keepdim=True) - n * (gw * n).mean(-1, keepdim=True)) * r
        out += [dx, (g * n).sum(0), g.sum(0)]
    return [v.to(dtype) for v in out]


def _plain_act(z, act):
    """(act(z), act'(z))."""
    if act == "none":
        return z, None
    if act == "relu":
        return z.clamp(min=0.0), (z > 0).float()
    if act == "silu":
        q = 1.0 / (1.0 + (-z).exp())
        return z * q, q * (1.0 + z * (1.0 - q))
    if act == "gelu":
        q = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * q, q + z * (-0.5 * z * z).exp() * (1.0 / math.sqrt(2.0 * math.pi))
    k = math.sqrt(2.0 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 0.134145 * z * z)


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    y, slope = _plain_act(x @ w.t() + s["bias"].float(), case["act"])
    out = [y + s["residual"].float() if case["residual"] else y]
    if case["step"]:
        g = s["g"].float()
        dz = g if slope is None else g * slope
        out += [dz @ w, dz.t() @ x, dz.sum(0)] + ([g] if case["residual"] else [])
    return [v.to(dtype) for v in out]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"clip": _plain_clip, "norm": _plain_norm, "linear": _plain_linear}[state["case"]["op"]](state)


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": n * e * (1 if case["inplace"] else 2), "flops": n * (2 if case["inplace"] else 3)}
    t, c, step = case["tokens"], case["cols"], case["step"]
    if case["op"] == "norm":
        # x, y, weight and bias; a step's g, dx and the two gradients more.
        return {"bytes": (t * c * (4 if step else 2) + c * (4 if step else 2)) * e, "flops": t * c * (20 if step else 8)}
    o = case["outs"]
    # x, weight, bias, y and the residual; a step's g and the gradients of all of them more.
    read = t * c + o * c + o + (t * o if case["residual"] else 0)
    moved = read + t * o + (read + t * o if step else 0)
    return {"bytes": moved * e, "flops": 2 * t * o * c * (3 if step else 1)}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_act(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(math.sqrt(8.0 / math.pi) * (z + 0.044715 * z**3))
    return z


def exact(case, seed):
    if case["op"] == "clip":
        grads = [g.double() for g in _inputs(case, seed)["grads"]]
        norm = torch.cat([torch.linalg.vector_norm(g).reshape(1) for g in grads]).norm()
        allowed = norm / case["factor"]
        factor = min(1.0, float(allowed / (norm + 1e-6)))
        return [norm.reshape(()), *[g * factor for g in grads]]
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    g = t.pop("g", None)
    args = [v.detach().requires_grad_(g is not None) for v in t.values()]
    if case["op"] == "norm":
        x, w, b = args
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = torch.addcmul(b, (x - mean) / torch.sqrt(var + _EPS), w)
    else:
        y = _exact_act(torch.addmm(args[2], args[0], args[1].t()), case["act"])
        y = y + args[3] if case["residual"] else y
    if g is None:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, args, g)]
