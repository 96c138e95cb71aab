"""nn.Linear with bias, activation and residual in its epilogue on the HIP path (csrc/linear_act.hip): the projections
and the feed-forward of the gated-linear-recurrence encoder layer."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}   # CRNN_ACT_* (include/crnn_hip.h)
_op = None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = act(x weight^T + bias) + residual for x [..., K] and weight [N, K] of one dtype (fp32, or bf16 on the bf16 matrix
    cores with fp32 accumulation), bias [N] in that dtype or fp32, residual [..., N] in that dtype (no broadcasting);
    activation "none", "relu", "gelu" (the erf form) or "silu". Bias, activation and residual are applied to the fp32 sums and
    y is rounded once. Differentiable once in every tensor: with an activation the backward keeps the pre-activation in x's
    dtype and rounds its gradient to it for the products with weight and x (bf16: d x and d weight are then good to about 2.4e-3
    in relative norm, where their own rounding is 1.7e-3); d weight and d bias come in their own dtypes from fp32 sums in a
    fixed order. Any sizes >= 1 and any strides: rows are read as they lie, except that the largest bf16 products copy rows
    that are not 16-byte aligned multiples of 8 elements into such ones first. weight, and each row of x, stays under 2 GiB.
    Runs on x's device and its current torch stream; capturable (a captured backward is refused while an eager graph of its
    leaves, built on the default stream, is alive). ValueError for arguments that do not fit, RuntimeError for CPU tensors and
    where it is traced (torch.compile, make_fx: torch.compiler.disable keeps it out) or differentiated by torch.func."""
    global _op
    if _op is None:
        _op = L.ops().linear.default
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return _op(x, weight, bias, act, residual)
