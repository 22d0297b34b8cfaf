"""Small batched matrix exponentials for PyTorch on AMD Instinct MI355X (gfx950)."""

import torch  # noqa: F401  (loads libc10/libtorch before the extension module)

from .ops.block import layer_norm, linear
from .ops.clip import clip_grad_norm, clip_grad_norm_, grad_norm
from .ops.hc_mix import mix_streams
from .ops.matrix_exp import matrix_exp, use_backend

__version__ = "0.1.0"
__all__ = [
    "clip_grad_norm",
    "clip_grad_norm_",
    "grad_norm",
    "layer_norm",
    "linear",
    "matrix_exp",
    "mix_streams",
    "use_backend",
]
