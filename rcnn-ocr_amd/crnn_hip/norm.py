"""Layer norm on the HIP path (csrc/layernorm.hip): the pre-norm of the gated-linear-recurrence encoder layer."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._lib import call_on, ptr


def _forward(x2, m: int, ldx: int, shape, weight, bias, eps: float, stats):
    y = torch.empty(shape, dtype=x2.dtype, device=x2.device)
    n = shape[-1]
    sp = ptr(stats)
    call_on(x2, "crnn_layernorm_fwd", L.dtype_code(x2.dtype), x2.data_ptr(), ldx, ptr(weight), ptr(bias), y.data_ptr(), n, sp,
            sp + 4 * m if stats is not None else None, m, n, eps)
    return y


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2, m, ldx = L.rows(x)
        n = x.shape[-1]
        stats = torch.empty(2 * m, dtype=torch.float32, device=x.device)   # mean, then rstd of every row
        y = _forward(x2, m, ldx, x.shape, weight, bias, eps, stats)
        ctx.save_for_backward(x2, weight, stats)
        ctx.geom = (x.shape, m, n, ldx, L.lib().crnn_layernorm_bwd_workspace(L.dtype_code(x.dtype), m, n))
        return y

    @staticmethod
    @L.differentiable_once
    def backward(ctx, dy):
        x2, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        shape, m, n, ldx, need = ctx.geom
        dy, _, ldd = L.rows(dy)
        dev = x2.device
        dx = torch.empty(shape, dtype=x2.dtype, device=dev) if need_x else None
        dw = torch.empty(n, dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty(n, dtype=torch.float32, device=dev) if need_b else None
        ws = torch.empty(need // 4, dtype=torch.float32, device=dev) if need_w or need_b else None
        sp = stats.data_ptr()
        call_on(x2, "crnn_layernorm_bwd", L.dtype_code(x2.dtype), dy.data_ptr(), ldd, x2.data_ptr(), ldx, ptr(weight), sp, sp + 4 * m,
                None, 0, ptr(dx), n, ptr(dw), ptr(db), 0, ptr(ws), need, m, n)
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
    if n > 1 << 30:
        raise ValueError(f"layer_norm: the last axis must be at most 2^30, got {n}")
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
    x2, m, ldx = L.rows(x)
    return _forward(x2, m, ldx, x.shape, weight, bias, float(eps), None)
