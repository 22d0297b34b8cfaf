"""The block between two stream mixings: layer norm and the linear layer with its epilogue.

``layer_norm(x, weight, bias, eps)`` normalises the last dimension; ``linear(x, weight, bias,
activation=..., residual=...)`` is ``activation(x @ weight.T + bias) + residual``.  Together they
make the generator of the mixing matrices from the normalised streams and the feed-forward block
that the mixed streams feed; the reference leaves both to the caller.

On a gfx950 device with float32 / float16 / bfloat16 operands of one type (weights of the norm and
the bias of the product may be float32 beside 16-bit operands) both run hand-written HIP kernels,
forward and backward.  Rows are read in place whatever their stride, so one stream of a
``[tokens, streams, width]`` tensor needs no copy.  Everything else -- CPU tensors, other types,
tensor subclasses, function transforms, forward-mode tangents, 2**31 rows or 2**30 columns of a norm,
2**30 rows or 2**22 columns or outputs of a product -- is composed from native PyTorch
operations, float16 and bfloat16 in float32; a backward that builds a graph takes differentiable
native pieces.
"""

from typing import Optional

import torch

from flash_hypercons import _C  # noqa: F401  (registers the flash_hypercons::* operators)
from flash_hypercons.ops.matrix_exp import _device_supported

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
# By name: the operator's code (FH_ACT_* of flash_hypercons.h) and the native composition.
_ACTIVATIONS = {
    None: (0, lambda z: z),
    "relu": (1, torch.nn.functional.relu),
    "gelu": (2, torch.nn.functional.gelu),
    "gelu_tanh": (3, lambda z: torch.nn.functional.gelu(z, approximate="tanh")),
    "silu": (4, torch.nn.functional.silu),
}
_NORM = torch.ops.flash_hypercons._layer_norm
_LINEAR = torch.ops.flash_hypercons._linear
# Rows and columns that the kernels take fewer than; a linear layer's outputs as its columns.
_NORM_ROWS, _NORM_COLS = 2**31, 2**30
_LINEAR_ROWS, _LINEAR_COLS = 2**30, 2**22


def _plain(t: Optional[torch.Tensor]) -> bool:
    return t is None or (
        type(t) in (torch.Tensor, torch.nn.Parameter)
        and t.device.type == "cuda"
        and t.layout == torch.strided
        and t.dtype in _DTYPES
        and torch.autograd.forward_ad.unpack_dual(t).tangent is None
    )


def _eligible(rows: int, cols: int, x: torch.Tensor, *others: Optional[torch.Tensor]) -> bool:
    """Operands for the HIP kernels, which check their shapes themselves; x has fewer rows and columns than these."""
    return (
        x is not None
        and _plain(x)
        and all(map(_plain, others))
        and torch.version.hip is not None
        and not torch._C._are_functorch_transforms_active()
        and x.ndim >= 1
        and 1 <= x.shape[-1] < cols
        and x.numel() // x.shape[-1] < rows
        and _device_supported(x.device.index)
    )


@torch.library.register_fake("flash_hypercons::_layer_norm")
def _layer_norm_fake(x, weight, bias, eps):
    return x.new_empty(x.shape)


@torch.library.register_fake("flash_hypercons::_layer_norm_forward")
def _layer_norm_forward_fake(x, weight, bias, eps):
    return x.new_empty(x.shape), x.new_empty((x.numel() // x.shape[-1], 2), dtype=torch.float32)


@torch.library.register_fake("flash_hypercons::_layer_norm_backward")
def _layer_norm_backward_fake(grad, x, weight, bias, stats, want_weight, want_bias):
    dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    cols = x.shape[-1]
    return (x.new_empty(x.shape), x.new_empty((cols if want_weight else 0,), dtype=dtype),
            x.new_empty((cols if want_bias else 0,), dtype=dtype))


@torch.library.register_fake("flash_hypercons::_linear")
def _linear_fake(x, weight, bias, residual, act):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.register_fake("flash_hypercons::_linear_forward")
def _linear_forward_fake(x, weight, bias, residual, act):
    rows = x.numel() // x.shape[-1] if act != 0 else 0
    saved = torch.float32 if x.dtype == torch.float32 else torch.float16
    return _linear_fake(x, weight, bias, residual, act), x.new_empty((rows, weight.shape[0]), dtype=saved)


@torch.library.register_fake("flash_hypercons::_linear_backward")
def _linear_backward_fake(grad, x, weight, bias, saved, act, want_x, want_weight, want_bias):
    return (x.new_empty(x.shape if want_x else (0,)), x.new_empty(weight.shape if want_weight else (0,)),
            x.new_empty((weight.shape[0] if want_bias else 0,), dtype=x.dtype if bias is None else bias.dtype))


def _wide(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """float16 and bfloat16 in float32, as the kernels compute them."""
    return t.float() if t is not None and t.dtype in (torch.float16, torch.bfloat16) else t


def layer_norm(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [..., C].

    weight and bias are [C] or None, of x's type or float32.  Differentiable in all three; the
    parameters' gradients are summed over the rows in a fixed order.
    """
    if _eligible(_NORM_ROWS, _NORM_COLS, x, weight, bias):
        return _NORM(x, weight, bias, eps)
    y = torch.nn.functional.layer_norm(_wide(x), x.shape[-1:], _wide(weight), _wide(bias), eps)
    return y.to(x.dtype)


def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    activation: Optional[str] = None,
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual for x [..., K] and weight [N, K].

    activation: None, "relu", "gelu" (by the error function), "gelu_tanh" or "silu"; bias: [N] of
    x's type or float32; residual: [..., N] of x's type, added after the activation.  Sums are
    float32 and rounded once.  Differentiable in every tensor.
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"linear: unknown activation {activation!r}; one of {', '.join(map(repr, _ACTIVATIONS))}")
    code, native = _ACTIVATIONS[activation]
    if (
        weight is not None
        and _eligible(_LINEAR_ROWS, _LINEAR_COLS, x, weight, bias, residual)
        and weight.ndim == 2
        and 1 <= weight.shape[0] < _LINEAR_COLS
    ):
        return _LINEAR(x, weight, bias, residual, code)
    y = native(torch.nn.functional.linear(_wide(x), _wide(weight), _wide(bias)))
    if residual is not None:
        if residual.shape != y.shape:
            raise ValueError(f"linear: expected a residual of shape {tuple(y.shape)}, got {tuple(residual.shape)}")
        y = y + _wide(residual)
    return y.to(x.dtype)


__all__ = ["layer_norm", "linear"]
