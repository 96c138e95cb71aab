"""The gated-linear-recurrence encoder, RCNN(rnn_type="glr"): a stack that takes the BiLSTM's place between the height
collapse and the head. The BiLSTM's steps are a dependent chain of matrix products; here the products over all frames come
first and only an element-wise recurrence runs along the line, so its time no longer grows with 2 T dependent steps.

One layer, x [B, T, H] (a first layer whose input has another width projects it first, `proj`):

    f, v = in(norm1(x)) [B, T, 2H each];  y = gated_scan(f, v, "both") [B, T, 2H];  x = x + out(y)
    x = x + ff2(gelu(ff1(norm2(x)))),  ff1: H -> 2H

run on the engine's workspace with the kernels behind crnn_hip.layer_norm, linear and gated_scan: norms and projections with
fp32 parameters' packed copies, the residuals in the products' epilogues, and in the backward the residual's gradient in
the norm's. Parameter gradients go straight into the parameters' fp32 .grad buffers.
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._lib import call, ptr
from .linear import ACTIVATIONS

EPS = 1e-5
BOTH = 2   # direction of crnn_gated_scan_fwd


def linears(eng, l):
    """(name, out features, in features) of layer l's products"""
    H = eng.H
    out = [("in", 4 * H, H), ("out", H, 2 * H), ("ff1", 2 * H, H), ("ff2", H, 2 * H)]
    if l == 0 and eng.enc_dim != H:
        out.insert(0, ("proj", H, eng.enc_dim))
    return out


class GLRStack:
    """forward / backward of the stack on a CRNNEngine's parameters, packed weights and workspace"""

    def __init__(self, engine):
        self.eng = engine

    # ---------------------------------------------------------------- pieces
    def _bytes(self, n):
        """scratch of one kernel call; the calls follow each other on one stream, so they share the largest asked for so far"""
        have = self.eng.ws.bufs.get("glr.ws")
        if n and (have is None or have.numel() < n):
            have = self.eng.ws.get("glr.ws", (n,), torch.uint8)
        return have if n else None

    def _norm(self, l, name, x, M, keep):
        e = self.eng
        pre = f"enc_rnn.{l}.{name}"
        y = e.ws.get(f"g{l}.{name}", (M, e.H), e.dtype)
        stats = e.ws.get(f"g{l}.{name}.stats", (2, M), torch.float32) if keep else None
        sp = ptr(stats)
        call("crnn_layernorm_fwd", e.dt, ptr(x), e.H, ptr(e.p[pre + ".weight"]), ptr(e.p[pre + ".bias"]), ptr(y), e.H, sp,
             sp + 4 * M if keep else None, M, e.H, EPS, L.stream_ptr())
        return y, stats

    def _norm_bwd(self, l, name, dy, x, stats, dres, dx, M, acc):
        e = self.eng
        pre = f"enc_rnn.{l}.{name}"
        need = L.lib().crnn_layernorm_bwd_workspace(e.dt, M, e.H)
        ws = self._bytes(need)
        sp = ptr(stats)
        call("crnn_layernorm_bwd", e.dt, ptr(dy), e.H, ptr(x), e.H, ptr(e.p[pre + ".weight"]), sp, sp + 4 * M, ptr(dres), e.H, ptr(dx),
             e.H, ptr(e._gview(pre + ".weight")), ptr(e._gview(pre + ".bias")), acc, ptr(ws), need, M, e.H, L.stream_ptr())

    def _linear(self, l, name, x, M, act="none", res=None, keep_z=False, y=None):
        e = self.eng
        pre = f"enc_rnn.{l}.{name}"
        w = e.packed[pre]
        n, k = w.shape
        a = ACTIVATIONS[act]
        y = e.ws.get(f"g{l}.{name}", (M, n), e.dtype) if y is None else y
        z = e.ws.get(f"g{l}.{name}.z", (M, n), e.dtype) if keep_z else None
        need = L.lib().crnn_linear_fwd_workspace(e.dt, ptr(x), k, ptr(w), k, M, n, k)
        ws = self._bytes(need)
        call("crnn_linear_fwd", e.dt, ptr(x), k, ptr(w), k, ptr(e.p[pre + ".bias"]), 1, a, ptr(res), n, ptr(y), n, ptr(z), n, ptr(ws), need,
             M, n, k, L.stream_ptr())
        return (y, z) if keep_z else y

    def _linear_bwd(self, l, name, dy, x, dx, M, acc, act="none", z=None):
        e = self.eng
        pre = f"enc_rnn.{l}.{name}"
        w = e.packed[pre]
        n, k = w.shape
        a = ACTIVATIONS[act]
        need = L.lib().crnn_linear_bwd_workspace(e.dt, ptr(dy), n, ptr(x), k, ptr(w), k, a, 1, 1, 1, M, n, k)
        ws = self._bytes(need)
        call("crnn_linear_bwd", e.dt, ptr(dy), n, ptr(x), k, ptr(w), k, ptr(z), n, a, ptr(dx), k, ptr(e._gview(pre + ".weight")), 1,
             ptr(e._gview(pre + ".bias")), 1, acc, ptr(ws), need, M, n, k, L.stream_ptr())

    # ---------------------------------------------------------------- the stack
    def forward(self, seq, B, T, keep):
        """seq [B, T, enc_dim] (compute dtype) -> (output [B, T, H], per-layer saved tensors)"""
        e = self.eng
        H, M, ws, lib = e.H, B * T, e.ws, L.lib()
        x, saved = seq, []
        for l in range(e.nl):
            s = {"in_": x}
            if l == 0 and e.enc_dim != H:
                x = self._linear(l, "proj", x, M)
            s["x"] = x
            s["n1"], s["st1"] = self._norm(l, "norm1", x, M, keep)
            s["u"] = u = self._linear(l, "in", s["n1"], M)   # [M][f forward | f reverse | v forward | v reverse]
            y = ws.get(f"g{l}.scan", (M, 2 * H), e.dtype)
            ckpt = None
            if keep:
                ckpt = ws.get(f"g{l}.ckpt", (lib.crnn_gated_scan_ckpt_bytes(e.dt, B, T, 2 * H, BOTH) // 4,), torch.float32)
            need = lib.crnn_gated_scan_workspace(e.dt, B, T, 2 * H, BOTH)
            w = self._bytes(need)
            call("crnn_gated_scan_fwd", e.dt, ptr(u), T * 4 * H, 4 * H, ptr(u[:, 2 * H:]), T * 4 * H, 4 * H, None, None, ptr(y), T * 2 * H,
                 2 * H, None, ptr(ckpt), ptr(w), need, B, T, 2 * H, BOTH, L.stream_ptr())
            s["y"], s["ckpt"] = y, ckpt
            s["x1"] = x = self._linear(l, "out", y, M, res=x)
            s["n2"], s["st2"] = self._norm(l, "norm2", x, M, keep)
            if keep:
                s["a"], s["z"] = self._linear(l, "ff1", s["n2"], M, act="gelu", keep_z=True)
            else:
                s["a"] = self._linear(l, "ff1", s["n2"], M, act="gelu")
            x = self._linear(l, "ff2", s["a"], M, res=x, y=ws.get(f"r{l}.out", (B, T, H), e.dtype))
            saved.append(s)
        return x, saved

    def backward(self, dx, saved, B, T, acc):
        """dx = d output [B, T, H] (compute dtype) -> d seq [B, T, enc_dim]; parameter gradients into the engine's grads"""
        e = self.eng
        H, M, ws, lib = e.H, B * T, e.ws, L.lib()
        buf = lambda name, n: ws.get("glr." + name, (M, n), e.dtype)  # noqa: E731
        d = dx
        for l in reversed(range(e.nl)):
            s = saved[l]
            da, dn = buf("da", 2 * H), buf("dn", H)
            self._linear_bwd(l, "ff2", d, s["a"], da, M, acc)
            self._linear_bwd(l, "ff1", da, s["n2"], dn, M, acc, act="gelu", z=s["z"])
            d1 = buf("d1", H)
            self._norm_bwd(l, "norm2", dn, s["x1"], s["st2"], d, d1, M, acc)
            self._linear_bwd(l, "out", d1, s["y"], da, M, acc)
            u, du = s["u"], buf("du", 4 * H)
            need = lib.crnn_gated_scan_workspace(e.dt, B, T, 2 * H, BOTH)
            w = self._bytes(need)
            call("crnn_gated_scan_bwd", e.dt, ptr(da), T * 2 * H, 2 * H, ptr(u), T * 4 * H, 4 * H, ptr(u[:, 2 * H:]), T * 4 * H, 4 * H, None,
                 None, ptr(s["ckpt"]), ptr(du), T * 4 * H, 4 * H, ptr(du[:, 2 * H:]), T * 4 * H, 4 * H, None, ptr(w), need, B, T, 2 * H, BOTH,
                 L.stream_ptr())
            self._linear_bwd(l, "in", du, s["n1"], dn, M, acc)
            d = buf(f"d0.{l % 2}", H)
            self._norm_bwd(l, "norm1", dn, s["x"], s["st1"], d1, d, M, acc)
            if l == 0 and e.enc_dim != H:
                dp = buf("dproj", e.enc_dim)
                self._linear_bwd(l, "proj", d, s["in_"], dp, M, acc)
                d = dp
        return d.view(B, T, -1)
