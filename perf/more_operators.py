"""Workloads of the two ends of a network of hyper-connected blocks, for timing and for checking results.

Two operators: ``embedding`` (rows of a table, scaled and copied into the residual streams, with the table's
gradient) and ``linear_cross_entropy`` (the softmax cross entropy of ``x @ weight.T + bias`` over a large
vocabulary, with its gradients).  Each runs forward alone (serving, scoring) or forward + gradients (training).

A case is a dict:

* ``op``: "embedding" or "loss"; ``dtype``; ``tokens``; ``vocab`` (rows of the table or of the weight); ``step``
  (gradients as well);
* embedding: ``cols``, ``streams`` (0: no dimension of streams), ``scaled`` (times sqrt(cols)), ``pad`` (the share
  of tokens that are padding, at the end of each sequence, left out of the gradient);
* loss: ``cols`` (of x), ``bias``, ``ignored`` (the share of positions without a target), ``reduction``.
"""

import math
import sys
from pathlib import Path

import torch

own = False  # True: the package's operators; False: plain torch operations in FP32

_ROOT = Path(__file__).resolve().parents[1]
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_PADDING = 0  # the table's row of the padding
_IGNORE = -100  # what stands where there is no target


def _package():
    path = str(_ROOT / "flash-hyperconnections_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_hypercons

    return flash_hypercons


def _embedding(name, dtype, tokens, cols, vocab, streams=0, scaled=False, pad=0.0, step=True):
    return {"name": name, "op": "embedding", "dtype": dtype, "tokens": tokens, "cols": cols, "vocab": vocab,
            "streams": streams, "scaled": scaled, "pad": pad, "step": step}


def _loss(name, dtype, tokens, cols, vocab, bias=False, ignored=0.0, reduction="mean", step=True):
    return {"name": name, "op": "loss", "dtype": dtype, "tokens": tokens, "cols": cols, "vocab": vocab, "bias": bias,
            "ignored": ignored, "reduction": reduction, "step": step}


def listed():
    return [
        # Serving: one token enters four residual streams.
        _embedding("emb_bf16_t1_c4096_s4", "bf16", 1, 4096, 131072, streams=4, step=False),
        # Training: a long batch enters four streams; the gradient fills a large table, most rows with zeros.
        _embedding("emb_bf16_t16384_c4096_v131072_s4_step", "bf16", 16384, 4096, 131072, streams=4),
        # Training of a small model on long sequences: few columns, many tokens, frequent ones by the thousand.
        _embedding("emb_f16_t131072_c512_v32768_scaled_step", "f16", 131072, 512, 32768, scaled=True),
        # A padded batch: nearly half the tokens are one row's.
        _embedding("emb_bf16_t8192_c2048_v65536_s2_pad_step", "bf16", 8192, 2048, 65536, streams=2, pad=0.45),
        # Single precision, a width that is no whole number of vectors, and an odd vocabulary.
        _embedding("emb_f32_t1500_c1027_v10007_scaled_step", "f32", 1500, 1027, 10007, scaled=True),
        # Scoring a single token: its negative logarithm of probability.
        _loss("loss_bf16_t1_c4096_v131072", "bf16", 1, 4096, 131072, reduction="none", step=False),
        # Scoring a batch's answers, each position by itself.
        _loss("loss_f16_t512_c2048_v65536", "f16", 512, 2048, 65536, reduction="none", step=False),
        # Training: a long batch over a large vocabulary; the largest.
        _loss("loss_bf16_t16384_c4096_v131072_step", "bf16", 16384, 4096, 131072),
        # Fine-tuning on answers: six positions in ten are prompts or padding, without a target.
        _loss("loss_bf16_t4096_c2048_v32768_ignored_step", "bf16", 4096, 2048, 32768, ignored=0.6),
        # A small batch whose positions are weighted by the caller.
        _loss("loss_f16_t200_c1024_v50001_bias_none_step", "f16", 200, 1024, 50001, bias=True, reduction="none"),
        # Single precision, odd sizes, a bias, a sum.
        _loss("loss_f32_t1500_c1027_v10007_bias_sum_step", "f32", 1500, 1027, 10007, bias=True, ignored=0.1,
              reduction="sum"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width over the logarithm of the range: whole vectors mostly, as models have, odd ones too."""
    w = _log_int(rng, low, high)
    return w if rng.random() < 0.35 or w < 64 else w - w % 64


def draw(rng):
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    vocab, step = _width(rng, 101, 131072), rng.random() < 0.7
    if rng.random() < 0.45:
        cols, streams = _width(rng, 33, 4096), rng.choice((0, 0, 1, 2, 4, 5))
        tokens = _log_int(rng, 1, min(131072, (1 << 28) // (cols * max(1, streams))))
        case = _embedding("", dtype, tokens, cols, vocab, streams, rng.random() < 0.5, rng.choice((0.0, 0.0, 0.4)), step)
    else:
        cols = _width(rng, 33, 4096)
        tokens = _log_int(rng, 1, max(1, min(16384, (1 << (36 if dtype == "f32" else 39)) // (cols * vocab))))
        case = _loss("", dtype, tokens, cols, vocab, rng.random() < 0.4, rng.choice((0.0, 0.0, 0.3)),
                     rng.choice(("mean", "mean", "sum", "none")), step)
    del case["name"]
    return case


def _words(count, vocab, gen):
    """Tokens as text has them: the n-th most frequent one about 1 / n as often as the first, which is word 1."""
    u = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.pow(float(vocab), u).long() % vocab).clamp_(0, vocab - 1)


def _inputs(case, seed):
    """The tensors of a case by name; "g" is the upstream gradient of a step."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    t, c, v = case["tokens"], case["cols"], case["vocab"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale)

    if case["op"] == "embedding":
        tokens = _words(t, v, gen)
        if case["pad"]:
            # Sequences of 128 positions, each with a tail of padding of its own length.
            at = torch.arange(t, device="cuda")
            share = torch.rand((t + 127) // 128, generator=gen, device="cuda") * (2 * case["pad"])
            tokens[at % 128 >= (128 * (1 - share))[at // 128]] = _PADDING
        got = {"tokens": tokens, "weight": normal(v, c, scale=c**-0.5).to(dtype)}
        if case["step"]:
            got["g"] = normal(*((t, case["streams"], c) if case["streams"] else (t, c)), scale=1e-2).to(dtype)
        return got
    weight = normal(v, c, scale=c**-0.5).to(dtype)
    targets = _words(t, v, gen)
    # Outputs of a network under training: anything between no idea of the target and near certainty.
    sure = torch.rand(t, 1, generator=gen, device="cuda").mul_(14.0)
    x = normal(t, c).addcmul_(weight[targets].float(), sure).to(dtype)
    got = {"x": x, "weight": weight}
    if case["bias"]:
        got["bias"] = normal(v, scale=0.5).to(dtype)
    if case["ignored"]:
        none = torch.rand(t, generator=gen, device="cuda") < case["ignored"]
        none[0] = False  # one has a target: the mean of none at all is no number
        targets[none] = _IGNORE
    got["targets"] = targets
    if case["step"]:
        # A weight for each position, or what a loss scaled for 16-bit gradients has upstream.
        got["g"] = normal(t).abs_() if case["reduction"] == "none" else torch.full((), 512.0, device="cuda")
    return got


def _scale(case):
    return math.sqrt(case["cols"]) if case["scaled"] else 1.0


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["step"]:
        state["args"] = [state[k].requires_grad_() for k in ("x", "weight", "bias") if k in state]
    return state


# ---- the package's operators ------------------------------------------------------------------


def _run_own(s):
    fh, case = _package(), s["case"]
    if case["op"] == "embedding":
        y = fh.embedding(s["tokens"], s["weight"], scale=_scale(case), streams=case["streams"] or None,
                         padding_idx=_PADDING if case["pad"] else None)
    else:
        y = fh.linear_cross_entropy(s["x"], s["weight"], s["targets"], s.get("bias"), ignore_index=_IGNORE,
                                    reduction=case["reduction"])
    return [y, *torch.autograd.grad(y, s["args"], s["g"])] if case["step"] else [y]


# ---- plain forms -------------------------------------------------------------------------------


def _plain_embedding(s):
    case, w, tokens = s["case"], s["weight"], s["tokens"]
    y = (w[tokens].float() * _scale(case)).to(w.dtype)
    if case["streams"]:
        y = y.unsqueeze(1).repeat(1, case["streams"], 1)
    if not case["step"]:
        return [y]
    g = s["g"].float()
    g = (g.sum(1) if case["streams"] else g) * _scale(case)
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, tokens, g)
    if case["pad"]:
        dw[_PADDING] = 0.0
    return [y, dw.to(w.dtype)]


def _plain_loss(s):
    case, dtype = s["case"], s["x"].dtype
    x, w, targets = s["x"].float(), s["weight"].float(), s["targets"]
    z = x @ w.t()
    if case["bias"]:
        z += s["bias"].float()
    valid = targets != _IGNORE
    at = targets.clamp(min=0).unsqueeze(1)
    m = z.amax(1, keepdim=True)
    chosen = z.gather(1, at)
    z = z.sub_(m).exp_()
    total = z.sum(1, keepdim=True)
    losses = torch.where(valid, (total.log() + (m - chosen)).squeeze(1), 0.0)
    count = valid.sum()
    out = [losses if case["reduction"] == "none" else losses.sum() / (count if case["reduction"] == "mean" else 1)]
    if case["step"]:
        g = s["g"] / count if case["reduction"] == "mean" else s["g"].expand(len(targets))
        dz = z.div_(total).scatter_add_(1, at, torch.full_like(chosen, -1.0))
        dz *= torch.where(valid, g, 0.0).unsqueeze(1)
        out += [(dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
        if case["bias"]:
            out.append(dz.sum(0).to(dtype))
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "loss": _plain_loss}[state["case"]["op"]](state)


def work(case):
    e = _BYTES[case["dtype"]]
    t, c, v, step = case["tokens"], case["cols"], case["vocab"], case["step"]
    if case["op"] == "embedding":
        # The tokens, their rows and the streams; a step's upstream gradient and the table's gradient more.
        n = max(1, case["streams"])
        bytes_ = 8 * t + (min(t, v) + t * n) * c * e + (8 * t + (t * n + v) * c * e if step else 0)
        return {"bytes": bytes_, "flops": t * c * (1 + n if step else 1)}
    # x, the weight, the bias, the targets and the losses; a step's gradients more.
    read = (t * c + v * c + (v if case["bias"] else 0)) * e
    losses = 4 * t if case["reduction"] == "none" else 4
    return {"bytes": (read + 8 * t + losses) * (2 if step else 1), "flops": (2 * t * v * c + 4 * t * v) * (3 if step else 1)}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_embedding(case, t):
    w = t["weight"].double()
    rows = torch.index_select(w, 0, t["tokens"]) * _scale(case)
    n = case["streams"]
    y = torch.stack([rows] * n, 1) if n else rows
    if not case["step"]:
        return [y]
    g = t["g"].double().reshape(case["tokens"], max(1, n), case["cols"]).sum(1)
    if case["pad"]:
        g[t["tokens"] == _PADDING] = 0.0
    # Sums over runs of sorted tokens, by differences of running sums in 64 bits within blocks of columns.
    order = torch.sort(t["tokens"], stable=True)
    dw = torch.zeros_like(w)
    words, lengths = torch.unique_consecutive(order.values, return_counts=True)
    ends = lengths.cumsum(0)
    for first in range(0, case["cols"], 256):
        run_sums = g[:, first : first + 256][order.indices].cumsum(0)[ends - 1]
        dw[words, first : first + 256] = torch.diff(run_sums, dim=0, prepend=torch.zeros_like(run_sums[:1]))
    return [y, dw * _scale(case)]


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(case, t)
    x, w = t["x"].double(), t["weight"].double()
    b = t["bias"].double() if case["bias"] else None
    targets, rows = t["targets"], case["tokens"]
    here = targets >= 0
    losses = torch.zeros(rows, dtype=torch.float64, device=x.device)
    upstream = None
    if case["step"]:
        upstream = t["g"].double().expand(rows) * here
        if case["reduction"] == "mean":
            upstream = upstream / here.sum()
    dx, dw = torch.zeros_like(x), torch.zeros_like(w) if case["step"] else None
    db = torch.zeros_like(b) if b is not None else None
    most = max(1, (1 << 28) // case["vocab"])
    for i in range(0, rows, most):
        part = slice(i, min(i + most, rows))
        z = x[part].mm(w.t())
        if b is not None:
            z += b
        logp = torch.log_softmax(z, 1)
        hit = here[part].nonzero().squeeze(1)
        losses[part][hit] = -logp[hit, targets[part][hit]]
        if case["step"]:
            p = logp.exp_()
            p[hit, targets[part][hit]] = torch.expm1(-losses[part][hit])
            p *= upstream[part, None]
            dx[part] = p.mm(w)
            dw.addmm_(p.t(), x[part])
            if db is not None:
                db += p.sum(0)
    if case["reduction"] == "none":
        out = [losses]
    else:
        out = [losses.sum() / (here.sum() if case["reduction"] == "mean" else 1)]
    return out + ([dx, dw] + ([db] if db is not None else []) if case["step"] else [])
