"""flash-train PyTorch binding: ``flash_train.torch.gemm``.

Same signature, checks and defaults as the reference binding
(python/flash_train/torch/csrc/flash_train_torch.cpp:34-75):
``gemm(a, b, c=None, alpha=1.0, beta=0.0) -> d`` with a (m x k), b (k x n)
and optional c (m x n) fp32, rank-2, contiguous device tensors; d is
allocated with ``torch.empty`` and computed on the current stream.
RuntimeError on any violated check.

Around a training step's products (include/flash_train/flash_train.h says
what each computes; none has a counterpart in the reference):
``linear_cross_entropy`` (an output head's loss, its logits never kept),
``moe_route`` (a router's choice, gates, packed rows and balance loss), both
differentiable and over their ``_forward`` and ``_backward`` calls, and
``clip_grad_norm``.

The native extension is required: importing this module without it raises
(there is no CPU or eager fallback).
"""

import ctypes
import os

import torch  # must load first: it brings the HIP runtime the library shares

_pkg = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ctypes.CDLL(os.path.join(_pkg, "libflash_train.so"), mode=ctypes.RTLD_GLOBAL)

try:
    from ._flash_train_torch import (  # noqa: E402
        clip_grad_norm,
        gemm,
        linear_cross_entropy_backward,
        linear_cross_entropy_forward,
        moe_route_backward,
        moe_route_forward,
    )
except ModuleNotFoundError as exc:  # pragma: no cover - build problem
    if exc.name != "flash_train.torch._flash_train_torch":
        raise
    raise RuntimeError(
        "flash_train.torch: the native extension is not built; run `python flash-train_amd/build.py`"
    ) from exc

from .training import linear_cross_entropy, moe_route  # noqa: E402

__all__ = [
    "gemm",
    "linear_cross_entropy",
    "linear_cross_entropy_forward",
    "linear_cross_entropy_backward",
    "moe_route",
    "moe_route_forward",
    "moe_route_backward",
    "clip_grad_norm",
]
