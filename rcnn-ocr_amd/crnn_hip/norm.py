"""Layer norm on the HIP path (csrc/layernorm.hip): the pre-norm of the gated-linear-recurrence encoder layer."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._lib import call_on, ptr


def layer_norm_fwd(x: torch.Tensor, weight, bias, eps: float, stats: bool):
    """-> (y, mean, rstd) of checked arguments; mean, rstd fp32 [rows] (None unless stats)"""
    x2, m, ldx = L.rows(x)
    n = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty(2, m, dtype=torch.float32, device=x.device)
    call_on(x, "crnn_layernorm_fwd", L.dtype_code(x.dtype), ptr(x2), ldx, ptr(weight), ptr(bias), ptr(y), n, ptr(mean),
            ptr(rstd), m, n, eps)
    return y, mean, rstd


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        n = x.shape[-1]
        x2, m, ldx = L.rows(x)
        dy2, _, ldd = L.rows(dy)
        dt = L.dtype_code(x.dtype)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty(n, dtype=torch.float32, device=x.device) if need_w else None
        db = torch.empty(n, dtype=torch.float32, device=x.device) if need_b else None
        ws, need = None, 0
        if need_w or need_b:
            need = L.lib().crnn_layernorm_bwd_workspace(dt, m, n)
            ws = torch.empty(need // 4, dtype=torch.float32, device=x.device)
        call_on(x, "crnn_layernorm_bwd", dt, ptr(dy2), ldd, ptr(x2), ldx, ptr(weight), ptr(mean), ptr(rstd), None, 0, ptr(dx), n,
                ptr(dw), ptr(db), 0, ptr(ws), need, m, n)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., N] (fp32 or bf16; var the population
    variance). weight, bias fp32 [N] (the encoder's parameters stay fp32), either may be None. Statistics and the weight
    gradients are fp32, y is rounded once to x's dtype. Differentiable once in x, weight and bias; the weight gradients
    add the rows in a fixed order. Runs on x's device and its current torch stream; capturable."""
    L.dtype_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x needs a last axis of at least one element, got {tuple(x.shape)}")
    n = x.shape[-1]
    if weight is not None:
        L.check_operand("layer_norm", "weight", weight, (n,), torch.float32, x.device)
        weight = weight.contiguous()
    if bias is not None:
        L.check_operand("layer_norm", "bias", bias, (n,), torch.float32, x.device)
        bias = bias.contiguous()
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    L.require_device(x)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return layer_norm_fwd(x, weight, bias, float(eps), False)[0]
