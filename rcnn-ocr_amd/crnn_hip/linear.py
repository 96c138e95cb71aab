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


def _forward(x2, m: int, ldx: int, shape, w2, ldw: int, bias, act: int, residual, z):
    n, k = w2.shape
    dt = L.dtype_code(x2.dtype)
    y = torch.empty(shape[:-1] + (n,), dtype=x2.dtype, device=x2.device)
    r2, ldr = None, n
    if residual is not None:
        r2, _, ldr = L.rows(residual)
    need = L.lib().crnn_linear_fwd_workspace(dt, x2.data_ptr(), ldx, w2.data_ptr(), ldw, m, n, k)
    ws = _bytes(need, x2.device)
    call_on(x2, "crnn_linear_fwd", dt, x2.data_ptr(), ldx, w2.data_ptr(), ldw, ptr(bias),
            1 if bias is not None and bias.dtype == torch.float32 else 0, act, ptr(r2), ldr, y.data_ptr(), n, ptr(z), n, ptr(ws), need,
            m, n, k)
    return y


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        x2, m, ldx = L.rows(x)
        w2, _, ldw = L.rows(weight)
        z = torch.empty(m, w2.shape[0], dtype=x.dtype, device=x.device) if act else None   # the pre-activation
        y = _forward(x2, m, ldx, x.shape, w2, ldw, bias, act, residual, z)
        ctx.save_for_backward(x2, w2, z)
        ctx.geom = (x.shape, m, ldx, ldw, act, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @L.differentiable_once
    def backward(ctx, dy):
        x2, w2, z = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        shape, m, ldx, ldw, act, bias_dtype = ctx.geom
        dx = dw = db = None
        if need_x or need_w or need_b:
            n, k = w2.shape
            dt = L.dtype_code(x2.dtype)
            dev = x2.device
            dy2, _, ldd = L.rows(dy)
            if need_x:
                dx = torch.empty(shape, dtype=x2.dtype, device=dev)
            if need_w:
                dw = torch.empty(n, k, dtype=w2.dtype, device=dev)
            if need_b:
                db = torch.empty(n, dtype=bias_dtype, device=dev)
            need = L.lib().crnn_linear_bwd_workspace(dt, dy2.data_ptr(), ldd, x2.data_ptr(), ldx, w2.data_ptr(), ldw, act, need_x,
                                                     need_w, need_b, m, n, k)
            ws = _bytes(need, dev)
            call_on(x2, "crnn_linear_bwd", dt, dy2.data_ptr(), ldd, x2.data_ptr(), ldx, w2.data_ptr(), ldw, ptr(z), n, act, ptr(dx), k,
                    ptr(dw), w2.dtype == torch.float32, ptr(db), bias_dtype == torch.float32, 0, ptr(ws), need, m, n, k)
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
    L.check_sizes("linear", *weight.shape)
    if bias is not None:
        L.check_operand("linear", "bias", bias, (n,), (x.dtype, torch.float32), x.device)
        bias = bias.contiguous()
    if residual is not None:
        L.check_operand("linear", "residual", residual, x.shape[:-1] + (n,), x.dtype, x.device)
    L.require_device(x)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LinearFn.apply(x, weight, bias, act, residual)
    x2, m, ldx = L.rows(x)
    w2, _, ldw = L.rows(weight)
    return _forward(x2, m, ldx, x.shape, w2, ldw, bias, act, residual, None)
