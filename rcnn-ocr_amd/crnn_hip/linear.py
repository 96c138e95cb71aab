"""nn.Linear with bias, activation and residual in its epilogue on the HIP path (csrc/linear_act.hip): the projections
and the feed-forward of the gated-linear-recurrence encoder layer."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._lib import call_on, ptr

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}   # CRNN_ACT_* (include/crnn_hip.h)


def _bytes(n: int, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def linear_fwd(x, weight, bias, act: int, residual, keep_z: bool):
    """-> (y, z) of checked arguments; z (the pre-activation, x's dtype) only if keep_z and there is an activation"""
    n, k = weight.shape
    dt = L.dtype_code(x.dtype)
    x2, m, ldx = L.rows(x)
    w2, _, ldw = L.rows(weight)
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    z = torch.empty(m, n, dtype=x.dtype, device=x.device) if keep_z and act else None
    r2, ldr = None, n
    if residual is not None:
        r2, _, ldr = L.rows(residual)
    need = L.lib().crnn_linear_fwd_workspace(dt, ptr(x2), ldx, ptr(w2), ldw, m, n, k)
    ws = _bytes(need, x.device)
    call_on(x, "crnn_linear_fwd", dt, ptr(x2), ldx, ptr(w2), ldw, ptr(bias),
            1 if bias is not None and bias.dtype == torch.float32 else 0, act, ptr(r2), ldr, ptr(y), n, ptr(z), n, ptr(ws), need,
            m, n, k)
    return y, z


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        y, z = linear_fwd(x, weight, bias, act, residual, True)
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            n, k = weight.shape
            dt = L.dtype_code(x.dtype)
            x2, m, ldx = L.rows(x)
            w2, _, ldw = L.rows(weight)
            dy2, _, ldd = L.rows(dy)
            if need_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            if need_w:
                dw = torch.empty(n, k, dtype=weight.dtype, device=x.device)
            if need_b:
                db = torch.empty(n, dtype=ctx.bias_dtype, device=x.device)
            need = L.lib().crnn_linear_bwd_workspace(dt, ptr(dy2), ldd, ptr(x2), ldx, ptr(w2), ldw, ctx.act, int(need_x),
                                                     int(need_w), int(need_b), m, n, k)
            ws = _bytes(need, x.device)
            call_on(x, "crnn_linear_bwd", dt, ptr(dy2), ldd, ptr(x2), ldx, ptr(w2), ldw, ptr(z), n, ctx.act, ptr(dx), k, ptr(dw),
                    int(weight.dtype == torch.float32), ptr(db), int(ctx.bias_dtype == torch.float32), 0, ptr(ws), need, m, n, k)
        return dx, dw, db, None, dy if need_r else None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = act(x weight^T + bias) + residual for x [..., K] and weight [N, K] of one dtype (fp32, or bf16 on the bf16 matrix
    cores with fp32 accumulation), bias [N] in that dtype or fp32, residual [..., N] in that dtype (no broadcasting);
    activation "none", "relu", "gelu" (the erf form) or "silu". Bias, activation and residual are applied to the fp32
    sums and y is rounded once. Differentiable once in every tensor: the backward keeps the pre-activation in x's dtype,
    d weight and d bias come in their own dtypes from fp32 sums in a fixed order. Any sizes >= 1 and any strides; rows that
    are not 16-byte aligned multiples of 8 elements are copied into such ones first. Runs on x's device and its current
    torch stream; capturable."""
    L.dtype_code(x.dtype)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1:
        raise ValueError("linear: x needs at least one axis")
    L.check_operand("linear", "weight", weight, None, x.dtype, x.device)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear: weight must be [N, {x.shape[-1]}] with N, K >= 1, got {tuple(weight.shape)}")
    n = weight.shape[0]
    if bias is not None:
        L.check_operand("linear", "bias", bias, (n,), (x.dtype, torch.float32), x.device)
        bias = bias.contiguous()
    if residual is not None:
        L.check_operand("linear", "residual", residual, x.shape[:-1] + (n,), x.dtype, x.device)
    L.require_device(x)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LinearFn.apply(x, weight, bias, act, residual)
    return linear_fwd(x, weight, bias, act, residual, False)[0]
