"""The global norm of many gradients, and clipping by it.

``grad_norm(tensors)`` is the norm of all elements of all tensors together.  ``clip_grad_norm``
returns new tensors scaled by ``min(1, max_norm / (norm + 1e-6))``; ``clip_grad_norm_`` scales the
gradients of parameters in place, as ``torch.nn.utils.clip_grad_norm_`` does, in two launches for
up to 96 tensors and two more for each further 96.

On a gfx950 device with float32 / float16 / bfloat16 tensors (of one device, types mixed as they
come) and a norm of 1, 2 or infinity, the HIP kernels run: sums are float64 and in one fixed order,
the norm is a float32 scalar on the device, and nothing waits for it.  Everything else, function
transforms and forward-mode tangents among it, is composed from native PyTorch operations.
"""

from typing import Iterable, List, Tuple, Union

import torch
from torch.autograd import forward_ad

from flash_hypercons import _C  # noqa: F401  (registers the flash_hypercons::* operators)
from flash_hypercons.ops.matrix_exp import _device_supported

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_TYPES = (1.0, 2.0, float("inf"))
_OPS = torch.ops.flash_hypercons
Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _eligible(tensors: List[torch.Tensor], norm_type: float) -> bool:
    if norm_type not in _TYPES or torch.version.hip is None or torch._C._are_functorch_transforms_active():
        return False
    device = tensors[0].device
    return (
        device.type == "cuda"
        and all(
            t.device == device and t.dtype in _DTYPES and t.layout == torch.strided
            and type(t) in (torch.Tensor, torch.nn.Parameter)
            for t in tensors
        )
        and (forward_ad._current_level < 0 or all(forward_ad.unpack_dual(t).tangent is None for t in tensors))
        and _device_supported(device.index)
    )


def _native_norm(tensors: List[torch.Tensor], norm_type: float) -> torch.Tensor:
    """In float64, which the factor of float64 gradients is made from; callers get it in float32."""
    device = tensors[0].device
    parts = [
        torch.linalg.vector_norm(t, norm_type, dtype=torch.complex128 if t.is_complex() else torch.float64).to(device)
        for t in tensors if t.numel()
    ]  # fmt: skip
    if not parts:
        return torch.zeros((), device=device, dtype=torch.float64)
    return torch.linalg.vector_norm(torch.stack(parts), norm_type)


def _factor(norm: torch.Tensor, max_norm: float) -> torch.Tensor:
    return (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _scaled(t: torch.Tensor, factor: torch.Tensor) -> torch.Tensor:
    if t.dtype in (torch.float64, torch.complex128):
        return t * factor.to(t.device)
    factor = factor.to(t.device, torch.float32)
    return t * factor if t.is_complex() else (t.float() * factor).to(t.dtype)


def _listed(tensors: Tensors) -> List[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


@torch.library.register_fake("flash_hypercons::_grad_norm")
def _grad_norm_fake(tensors, norm_type):
    return tensors[0].new_empty((), dtype=torch.float32)


@torch.library.register_fake("flash_hypercons::_clip_grads")
def _clip_grads_fake(tensors, max_norm, norm_type):
    # Dense tensors keep their strides, and the others' results are contiguous.
    dense = torch.ops.aten.is_non_overlapping_and_dense
    clipped = [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device)
               if not t.is_neg() and dense(t) else t.new_empty(t.shape) for t in tensors]
    return clipped, tensors[0].new_empty((), dtype=torch.float32)


@torch.library.register_fake("flash_hypercons::_clip_grads_")
def _clip_grads_inplace_fake(tensors, max_norm, norm_type):
    return tensors[0].new_empty((), dtype=torch.float32)


@torch.no_grad()
def grad_norm(tensors: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of `tensors` together: a float32 scalar; 0 without tensors."""
    listed, norm_type = _listed(tensors), float(norm_type)
    if not listed:
        return torch.zeros(())
    return _OPS._grad_norm(listed, norm_type) if _eligible(listed, norm_type) else _native_norm(listed, norm_type).float()


@torch.no_grad()
def clip_grad_norm(
    tensors: Tensors, max_norm: float, norm_type: float = 2.0
) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """New tensors, `tensors` times min(1, max_norm / (norm + 1e-6)), and the norm."""
    listed, max_norm, norm_type = _listed(tensors), float(max_norm), float(norm_type)
    if not listed:
        return [], torch.zeros(())
    if _eligible(listed, norm_type):
        return _OPS._clip_grads(listed, max_norm, norm_type)
    norm = _native_norm(listed, norm_type)
    factor = _factor(norm, max_norm)
    return [_scaled(t, factor) for t in listed], norm.float()


@torch.no_grad()
def clip_grad_norm_(
    parameters: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False
) -> torch.Tensor:
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)); returns the norm.

    Parameters without a gradient are left out; gradients that the norm allows stay as they are.
    Where the HIP kernels run, dense gradients that share memory (one listed twice among them) raise
    before anything is scaled; composed natively, as in torch, each mention scales the memory again.
    Gradients with gaps are copied and not compared.
    ``error_if_nonfinite`` raises before anything is scaled, and waits for the norm to do so.
    """
    grads = [p.grad for p in _listed(parameters) if p.grad is not None]
    max_norm, norm_type = float(max_norm), float(norm_type)
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"the global norm of order {norm_type} of the gradients is {norm.item()}")
    if _eligible(grads, norm_type):
        return _OPS._clip_grads_(grads, max_norm, norm_type)
    norm = _native_norm(grads, norm_type)
    factor = _factor(norm, max_norm)
    for g in grads:
        g.copy_(_scaled(g, factor))
    return norm.float()


__all__ = ["clip_grad_norm", "clip_grad_norm_", "grad_norm"]
