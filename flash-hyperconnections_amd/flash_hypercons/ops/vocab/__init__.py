"""The two ends of a network of hyper-connected blocks: the embedding and the loss over the vocabulary.

``embedding(tokens, weight, scale=..., streams=n)`` looks rows of a table up, scales them and copies them
into the n residual streams; ``linear_cross_entropy(x, weight, targets, bias)`` is the softmax cross entropy
of ``x @ weight.T + bias``, whose logits are never kept.  The reference leaves both to the caller.

On a gfx950 device with float32 / float16 / bfloat16 operands of one type (the bias may be float32 beside
16-bit operands) and int64 or int32 indices both run hand-written HIP kernels, forward and backward.
Everything else -- CPU tensors, other types, tensor subclasses, function transforms, forward-mode tangents,
2**28 tokens or rows of a table, 2**24 of its columns, 2**16 streams; 2**24 rows of x, 2**22 columns
or words -- is composed from native PyTorch operations, float16 and bfloat16 in float32; a backward that
builds a graph takes differentiable native pieces.

An index that is out of range raises on the CPU.  On the GPU nothing waits to find out: such a token's
row, or such a target's loss, is NaN, and so are the gradients that the loss reaches; the embedding's
gradient leaves such a token out.
"""

from typing import Optional

import torch

from flash_hypercons import _C  # noqa: F401  (registers the flash_hypercons::* operators)
from flash_hypercons.ops.block import _plain, _wide
from flash_hypercons.ops.matrix_exp import _device_supported

_INDICES = (torch.int64, torch.int32)
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # FH_REDUCE_* of flash_hypercons.h
_EMBEDDING = torch.ops.flash_hypercons._embedding
_LOSS = torch.ops.flash_hypercons._linear_cross_entropy
# What the kernels take fewer of.
_TOKENS, _TABLE_ROWS, _TABLE_COLS, _STREAMS = 2**28, 2**28, 2**24, 2**16
_LOSS_ROWS, _LOSS_COLS = 2**24, 2**22


def _eligible(indices: torch.Tensor, *operands: Optional[torch.Tensor]) -> bool:
    """Tensors for the HIP kernels, which check their shapes themselves."""
    return (
        type(indices) in (torch.Tensor, torch.nn.Parameter)
        and indices.device.type == "cuda"
        and indices.layout == torch.strided
        and indices.dtype in _INDICES
        and all(map(_plain, operands))
        and torch.version.hip is not None
        and not torch._C._are_functorch_transforms_active()
        and _device_supported(indices.device.index)
    )


def _in_range(indices: torch.Tensor, count: int) -> torch.Tensor:
    """Which indices on the GPU are in 0 .. count - 1: PyTorch reads memory at the others without a check."""
    if count == 0 and indices.numel():
        raise IndexError("no index is in the range of a table with no rows")
    return (indices >= 0) & (indices < count)


@torch.library.register_fake("flash_hypercons::_embedding")
def _embedding_fake(tokens, weight, scale, streams, padding):
    return weight.new_empty((*tokens.shape, *((streams,) if streams else ()), weight.shape[1]))


@torch.library.register_fake("flash_hypercons::_embedding_backward")
def _embedding_backward_fake(grad, tokens, vocab, scale, streams, padding):
    return grad.new_empty((vocab, grad.shape[-1]))


@torch.library.register_fake("flash_hypercons::_linear_cross_entropy")
def _linear_cross_entropy_fake(x, weight, targets, bias, ignore, reduction):
    return x.new_empty(targets.shape if reduction == 0 else (), dtype=torch.float32)


@torch.library.register_fake("flash_hypercons::_linear_cross_entropy_forward")
def _linear_cross_entropy_forward_fake(x, weight, targets, bias, ignore, reduction):
    loss = _linear_cross_entropy_fake(x, weight, targets, bias, ignore, reduction)
    return loss, x.new_empty((x.numel() // x.shape[-1], 2), dtype=torch.float32)


@torch.library.register_fake("flash_hypercons::_linear_cross_entropy_backward")
def _linear_cross_entropy_backward_fake(grad, x, weight, targets, bias, lse, ignore, reduction, want_x, want_weight,
                                        want_bias):
    return (x.new_empty(x.shape if want_x else (0,)), x.new_empty(weight.shape if want_weight else (0,)),
            x.new_empty((weight.shape[0] if want_bias else 0,), dtype=x.dtype if bias is None else bias.dtype))


@torch.library.register_fake("flash_hypercons::_linear_cross_entropy_ahead")
def _linear_cross_entropy_ahead_fake(x, weight, targets, bias, ignore, reduction, want_x, want_weight, want_bias):
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]

    def sums(want, *shape):
        return x.new_empty(shape if want else (0,), dtype=torch.float32)

    return (sums(True), x.new_empty((rows + 1,), dtype=torch.int32), sums(want_x, rows, cols),
            sums(want_weight, weight.shape[0], cols), sums(want_bias, weight.shape[0]))


@torch.library.register_fake("flash_hypercons::_linear_cross_entropy_scale")
def _linear_cross_entropy_scale_fake(grad, x, weight, targets, bias, places, dx_sums, dw_sums, db_sums, ignore,
                                     reduction):
    return (x.new_empty(x.shape if dx_sums.numel() else (0,)), x.new_empty(weight.shape if dw_sums.numel() else (0,)),
            x.new_empty((weight.shape[0] if db_sums.numel() else 0,), dtype=x.dtype if bias is None else bias.dtype))


def embedding(
    tokens: torch.Tensor,
    weight: torch.Tensor,
    *,
    scale: float = 1.0,
    streams: Optional[int] = None,
    padding_idx: Optional[int] = None,
) -> torch.Tensor:
    """scale * weight[tokens], copied into `streams` residual streams: [*tokens, C], or [*tokens, streams, C].

    tokens: int64 or int32, of any shape; weight: [V, C].  Differentiable in weight: a row's gradient is
    the sum over the places of its token, in their order, and over the streams, in float32 and rounded once.
    The row `padding_idx` (from the end where negative) has a gradient of zero.
    """
    if streams is not None and streams < 1:
        raise ValueError(f"embedding: expected a positive number of streams, got {streams}")
    if weight.ndim != 2:
        raise ValueError(f"embedding: expected weight [V, C], got {tuple(weight.shape)}")
    vocab, cols = weight.shape
    if padding_idx is not None:
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"embedding: padding_idx {padding_idx} is not a row of {vocab}")
        padding_idx %= vocab
    if (
        _eligible(tokens, weight)
        and tokens.numel() < _TOKENS
        and 1 <= vocab < _TABLE_ROWS
        and 1 <= cols < _TABLE_COLS
        and (streams or 1) < _STREAMS
    ):
        return _EMBEDDING(tokens, weight, scale, streams or 0, -1 if padding_idx is None else padding_idx)
    if tokens.device.type == "cuda":
        valid = _in_range(tokens, vocab)
        y = torch.nn.functional.embedding(torch.where(valid, tokens, 0), _wide(weight), padding_idx) * scale
        y = torch.where(valid.unsqueeze(-1), y, float("nan"))
    else:
        y = torch.nn.functional.embedding(tokens, _wide(weight), padding_idx) * scale
    if streams is not None:
        y = y.unsqueeze(-2).expand(*tokens.shape, streams, cols)
    return y.to(weight.dtype).contiguous()


def linear_cross_entropy(
    x: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """The softmax cross entropy of x @ weight.T + bias for x [..., K], weight [V, K] and targets [...].

    bias: [V] of x's type or float32.  The logits are formed in pieces, in float32, and never kept.  Where
    a gradient is wanted of a sum or mean over 1024 positions or more (128 in float32), the gradients are
    formed with the loss, as float32 sums that the backward scales by the upstream gradient; otherwise the
    backward forms the logits again.  Losses are float32 (float64 for float64 operands): of each position for
    reduction "none", else their "sum", or their "mean" over the positions with a target (NaN where there
    is none).  A position whose target is `ignore_index` has a loss and gradients of zero, whatever x holds
    there, and costs next to nothing.  Differentiable in x, weight and bias.

    What 16 bits cost beside float32 products rounded once: exponentials come from the hardware's exp2; where
    gradients are formed with the loss they wait for their row's sum in float16, 11 bits each; and the
    logits' gradients are rounded to x's type before they are multiplied, with batches of up to 128 positions
    to twice its digits.  The batch's size decides, not how many positions have a target.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: unknown reduction {reduction!r}; one of {', '.join(map(repr, _REDUCTIONS))}")
    if (
        _eligible(targets, x, weight, bias)
        and x.ndim >= 1
        and weight.ndim == 2
        and 1 <= x.shape[-1] < _LOSS_COLS
        and x.numel() // x.shape[-1] < _LOSS_ROWS
        and 1 <= weight.shape[0] < _LOSS_COLS
    ):
        return _LOSS(x, weight, targets, bias, ignore_index, _REDUCTIONS[reduction])
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: expected targets of shape {tuple(x.shape[:-1])}, got {tuple(targets.shape)}")
    rows = _wide(x).reshape(-1, x.shape[-1])
    flat = targets.reshape(-1).long()
    here = flat != ignore_index
    # What a position without a target holds takes no part, a NaN among it.
    rows = torch.where(here.unsqueeze(1), rows, rows.new_zeros(()))
    valid = None
    if flat.device.type == "cuda":
        valid = _in_range(flat, weight.shape[0])
        # The row's logits are NaN then, and its gradients too.
        rows = rows + torch.where(here & ~valid, float("nan"), 0.0).to(rows.dtype).unsqueeze(1)
    z = torch.nn.functional.linear(rows, _wide(weight), _wide(bias))
    if valid is not None:
        loss = torch.nn.functional.cross_entropy(z, torch.where(valid, flat, 0), reduction="none")
        loss = torch.where(here, loss, 0.0)
        if reduction != "none":
            loss = loss.sum() / (here.sum() if reduction == "mean" else 1)
    else:
        loss = torch.nn.functional.cross_entropy(z, flat, ignore_index=ignore_index, reduction=reduction)
    return loss.reshape(targets.shape) if reduction == "none" else loss


__all__ = ["embedding", "linear_cross_entropy"]
