"""Gated linear recurrence along a sequence on the HIP path (csrc/scan.hip): the mixer of the gated-linear-recurrence
encoder layer, beside the BiLSTM sweeps (csrc/lstm_seq.hip). Unlike the LSTM's, its steps compose, so a long sequence is
cut and its pieces run at once."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._lib import call_on, ptr

DIRECTIONS = {"forward": 0, "reverse": 1, "both": 2}   # `dir` of crnn_gated_scan_fwd (include/crnn_hip.h)


def _chan(t: torch.Tensor) -> torch.Tensor:
    """channels contiguous"""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _floats(nbytes: int, device):
    return torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None


def _forward(f, v, h0, lengths, direction: int, need: int, hT, ckpt):
    """y of checked [B, T, D] arguments, channels contiguous; hT and ckpt (each may be None) are written"""
    B, T, D = f.shape
    y = torch.empty(B, T, D, dtype=f.dtype, device=f.device)
    ws = _floats(need, f.device)
    fs, vs = f.stride(), v.stride()
    call_on(f, "crnn_gated_scan_fwd", L.dtype_code(f.dtype), f.data_ptr(), fs[0], fs[1], v.data_ptr(), vs[0], vs[1], ptr(h0), ptr(lengths),
            y.data_ptr(), T * D, D, ptr(hT), ptr(ckpt), ptr(ws), need, B, T, D, direction)
    return y


class _GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, v, h0, lengths, direction, want_state):
        B, T, D = f.shape
        dt = L.dtype_code(f.dtype)
        lib = L.lib()
        f, v = _chan(f), _chan(v)
        need = lib.crnn_gated_scan_workspace(dt, B, T, D, direction)
        ckpt = _floats(lib.crnn_gated_scan_ckpt_bytes(dt, B, T, D, direction), f.device)   # what the backward starts from
        hT = torch.empty(B, D, dtype=torch.float32, device=f.device) if want_state else None
        y = _forward(f, v, h0, lengths, direction, need, hT, ckpt)
        ctx.save_for_backward(f, v, lengths, ckpt)
        ctx.geom = (direction, need)
        ctx.set_materialize_grads(False)
        return (y, hT) if want_state else y

    @staticmethod
    @L.differentiable_once
    def backward(ctx, dy, dhT=None):
        f, v, lengths, ckpt = ctx.saved_tensors
        need_f, need_v, need_h, _, _, _ = ctx.needs_input_grad
        direction, need = ctx.geom
        B, T, D = f.shape
        dev = f.device
        # only the final state was used: no upstream gradient for y
        dy = torch.zeros(B, T, D, dtype=f.dtype, device=dev) if dy is None else _chan(dy)
        if dhT is not None:
            dhT = dhT.contiguous()
        df = torch.empty(B, T, D, dtype=f.dtype, device=dev)
        dv = torch.empty(B, T, D, dtype=f.dtype, device=dev)
        dh0 = torch.empty(B, D, dtype=torch.float32, device=dev) if need_h else None
        ws = _floats(need, dev)
        fs, vs, ds = f.stride(), v.stride(), dy.stride()
        call_on(f, "crnn_gated_scan_bwd", L.dtype_code(f.dtype), dy.data_ptr(), ds[0], ds[1], f.data_ptr(), fs[0], fs[1], v.data_ptr(), vs[0],
                vs[1], ptr(lengths), ptr(dhT), ptr(ckpt), df.data_ptr(), T * D, D, dv.data_ptr(), T * D, D, ptr(dh0), ptr(ws), need, B, T, D,
                direction)
        return df if need_f else None, dv if need_v else None, dh0, None, None, None


def _infer(f, v, h0, lengths, direction: int, hT):
    f, v = _chan(f), _chan(v)
    return _forward(f, v, h0, lengths, direction, L.lib().crnn_gated_scan_workspace(L.dtype_code(f.dtype), *f.shape, direction), hT, None)


def gated_scan(f: torch.Tensor, v: torch.Tensor, h0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
               direction: str = "forward", return_state: bool = False):
    """h_t = a_t h_{t-1} + (1 - a_t) v_t with a_t = sigmoid(f_t), per channel, for gate logits f and values v [B, T, D] (fp32 or
    bf16); -> y [B, T, D] with y_t = h_t in their dtype, the state in fp32 throughout. f, v may be strided views (the two
    halves of one projection). direction "forward" (t = 0 ..), "reverse" (from the last step back) or "both" (channels
    [0, D/2) forward, [D/2, D) in reverse, as the BiLSTM lays its directions out; D even).
    h0 fp32 [B, D]: the state before the first step walked (None: 0). lengths int32 / int64 [B] (None: all T): steps at or behind
    lengths[b] (clamped to 0 .. T) are not read, get y = 0 and no gradient, and leave the state as it is.
    return_state: -> (y, hT), hT fp32 [B, D] the state after the last step walked, from which the next stretch of the
    sequence continues. Differentiable once in f, v and h0. Runs on f's device and its current torch stream; capturable
    where lengths is an int32 tensor on the device (another one is converted)."""
    L.dtype_code(f.dtype)
    dr = DIRECTIONS.get(direction)
    if dr is None:
        raise ValueError(f"gated_scan: direction must be one of {sorted(DIRECTIONS)}, got {direction!r}")
    if f.dim() != 3:
        raise ValueError(f"gated_scan: f must be [B, T, D], got {tuple(f.shape)}")
    L.check_operand("gated_scan", "v", v, f.shape, f.dtype, f.device)
    B, T, D = f.shape
    L.check_sizes("gated_scan", B, T, D)
    if dr == 2 and D % 2:
        raise ValueError(f"gated_scan: direction 'both' needs an even number of channels, got {D}")
    if h0 is not None:
        L.check_operand("gated_scan", "h0", h0, (B, D), torch.float32, f.device)
        h0 = h0.contiguous()
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"gated_scan: lengths must be an int32 or int64 tensor of shape ({B},)")
    L.require_device(f)
    if lengths is not None:
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, T)   # before the conversion: a value past 32 bits must not wrap
        lengths = lengths.to(device=f.device, dtype=torch.int32).contiguous()
    if torch.is_grad_enabled() and (f.requires_grad or v.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScanFn.apply(f, v, h0, lengths, dr, return_state)
    hT = torch.empty(B, D, dtype=torch.float32, device=f.device) if return_state else None
    y = _infer(f, v, h0, lengths, dr, hT)
    return (y, hT) if return_state else y


def gated_scan_step(f: torch.Tensor, v: torch.Tensor, state: torch.Tensor, out_state: Optional[torch.Tensor] = None):
    """one step of running sequences: f, v [B, D] (fp32 or bf16), state fp32 [B, D] -> (y [B, D], next state). out_state: where the
    next state is written (fp32 [B, D], contiguous); `state` itself updates it in place. Inference only."""
    L.dtype_code(f.dtype)
    if f.dim() != 2:
        raise ValueError(f"gated_scan_step: f must be [B, D], got {tuple(f.shape)}")
    L.check_sizes("gated_scan_step", *f.shape)
    L.check_operand("gated_scan_step", "v", v, f.shape, f.dtype, f.device)
    L.check_operand("gated_scan_step", "state", state, f.shape, torch.float32, f.device)
    if torch.is_grad_enabled() and (f.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError("gated_scan_step is inference only: use gated_scan(..., return_state=True) where gradients are needed")
    if out_state is not None:
        L.check_operand("gated_scan_step", "out_state", out_state, f.shape, torch.float32, f.device)
        if not out_state.is_contiguous():
            raise ValueError("gated_scan_step: out_state must be contiguous")
        a, b, n = out_state.data_ptr(), state.data_ptr(), 4 * out_state.numel()
        same = a == b and state.is_contiguous()
        span = 4 * (sum((s - 1) * st for s, st in zip(state.shape, state.stride())) + 1) if state.numel() else 0
        if not same and a < b + span and b < a + n:
            raise ValueError("gated_scan_step: out_state overlaps state without being it")
    L.require_device(f)
    if out_state is None:
        out_state = torch.empty(f.shape, dtype=torch.float32, device=f.device)
    y = _infer(f.unsqueeze(1), v.unsqueeze(1), state.contiguous(), None, 0, out_state)
    return y.squeeze(1), out_state
