"""Layer norm on the HIP path (csrc/layernorm.hip): the pre-norm of the gated-linear-recurrence encoder layer."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

_op = None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., N] (fp32 or bf16; var the population
    variance). weight, bias fp32 [N] (the encoder's parameters stay fp32), either may be None. Statistics and the weight
    gradients are fp32, y is rounded once to x's dtype. Differentiable once in x, weight and bias; the weight gradients add
    the rows in a fixed order. Runs on x's device and its current torch stream; capturable (a captured backward is refused
    while an eager graph of its leaves, built on the default stream, is alive). ValueError for arguments that do not fit,
    RuntimeError for CPU tensors and where it is traced (torch.compile, make_fx: torch.compiler.disable keeps it out) or
    differentiated by torch.func."""
    global _op
    if _op is None:
        _op = L.ops().layer_norm.default
    return _op(x, weight, bias, eps)
