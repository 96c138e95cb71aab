"""Gated linear recurrence along a sequence on the HIP path (csrc/scan.hip): the mixer of the gated-linear-recurrence
encoder layer, beside the BiLSTM sweeps (csrc/lstm_seq.hip). Unlike the LSTM's, its steps compose, so a long sequence is
cut and its pieces run at once."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

DIRECTIONS = {"forward": 0, "reverse": 1, "both": 2}   # `dir` of crnn_gated_scan_fwd (include/crnn_hip.h)
_op = None


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
    where lengths is an int32 tensor on the device (another one is converted); a captured backward is refused while an eager
    graph of its leaves, built on the default stream, is alive. ValueError for arguments that do not fit,
    RuntimeError for CPU tensors and where it is traced (torch.compile, make_fx: torch.compiler.disable keeps it out) or
    differentiated by torch.func."""
    global _op
    if _op is None:
        _op = L.ops().gated_scan.default
    dr = DIRECTIONS.get(direction)
    if dr is None:
        raise ValueError(f"gated_scan: direction must be one of {sorted(DIRECTIONS)}, got {direction!r}")
    if lengths is not None and not isinstance(lengths, torch.Tensor):
        raise ValueError(f"gated_scan: lengths must be an int32 or int64 tensor, got {type(lengths).__name__}")
    out = _op(f, v, h0, lengths, dr, return_state)
    return out if return_state else out[0]


def gated_scan_step(f: torch.Tensor, v: torch.Tensor, state: torch.Tensor, out_state: Optional[torch.Tensor] = None):
    """one step of running sequences: f, v [B, D] (fp32 or bf16), state fp32 [B, D] -> (y [B, D], next state). out_state: where the
    next state is written (fp32 [B, D], contiguous, over none of the inputs); `state` itself updates it in place. Inference
    only."""
    return L.ops().gated_scan_step.default(f, v, state, out_state)
