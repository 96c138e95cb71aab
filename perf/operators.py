"""Timing cases of the sequence operators that make up a gated-linear-recurrence encoder layer:

  layer_norm   y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis
  linear       y = act(x W^T + bias) + residual
  gated_scan   h_t = a_t h_{t-1} + (1 - a_t) v_t with a_t = sigmoid(f_t), along the sequence

each as inference (forward only) and as a training pass (forward, then every gradient). `run` computes a case either
in its plain form (elementary torch operations in fp32) or, where `own` is true, through crnn_hip's operators on the
same state; `exact` evaluates the definitions in fp64.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def _ln(name, rows, n, dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "n": n, "dtype": dtype, "train": train}


def _lin(name, rows, k, n, dtype, train, act, bias, res):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "train": train, "act": act,
            "bias": bias, "res": res}


def _scan(name, b, t, d, dtype, train, direction, ragged, state):
    return {"name": name, "op": "gated_scan", "b": b, "t": t, "d": d, "dtype": dtype, "train": train,
            "direction": direction, "ragged": ragged, "state": state}


def listed():
    return [
        # one 32 x 128 line at inference: 16 frames of a 512-wide encoder, launch latency
        _ln("ln one line", 16, 512, "bf16", False),
        # the training batch: 256 lines of 32 frames (32 x 256 crops), hidden 512
        _ln("ln train batch", 8192, 512, "bf16", True),
        # an odd width whose rows are not 16-byte aligned, exact-fp32 parity mode
        _ln("ln ragged fp32", 1999, 1021, "fp32", True),
        # long lines (32 x 1024 crops, 128 frames) at batch 512, hidden 768
        _ln("ln long lines", 65536, 768, "bf16", True),
        # one line through the feed-forward's first half
        _lin("linear one line", 16, 512, 1024, "bf16", False, "gelu", True, False),
        # the training batch through the feed-forward's first half
        _lin("linear train batch", 8192, 512, 1024, "bf16", True, "gelu", True, False),
        # odd sizes in the exact-fp32 parity mode
        _lin("linear ragged fp32", 1027, 509, 1021, "fp32", True, "silu", True, True),
        # long lines at batch 256 through the feed-forward's second half, closing the residual branch
        _lin("linear long lines", 32768, 1536, 768, "bf16", True, "none", True, True),
        # streaming: the next frame of 64 running lines, state carried between calls
        _scan("scan next frame", 64, 1, 1024, "bf16", False, "forward", False, True),
        # the training batch, both directions (hidden 512 each), as the bidirectional encoder runs it
        _scan("scan train batch", 256, 32, 1024, "bf16", True, "both", False, False),
        # lines of different lengths (an empty one and a one-frame one among them), odd sizes, exact-fp32 parity mode
        _scan("scan ragged fp32", 37, 301, 333, "fp32", True, "reverse", True, True),
        # few but very long sequences
        _scan("scan long", 2, 16384, 1024, "bf16", True, "forward", False, True),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    """the ranges: 1 .. 65536 rows of 16 .. 4096 columns (layer norm); 1 .. 32768 rows, 8 .. 2048 wide on both sides
    (linear); 1 .. 256 sequences of 1 .. 16384 steps, 2 .. 1536 channels (scan). Half of the sizes are rounded to a
    multiple of 64, the rest are as they fall; each within the work of the largest listed case of its operator."""
    def size(lo, hi):
        n = _log_int(rng, lo, hi)
        if n >= 64 and rng.random() < 0.5:
            n = n // 64 * 64
        return n

    op = rng.choice(["layer_norm", "linear", "gated_scan"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    train = rng.random() < 0.6
    while True:
        if op == "layer_norm":
            c = _ln("", size(1, 65536), size(16, 4096), dtype, train)
            if c["rows"] * c["n"] * (1 if dtype == "bf16" else 2) > 65536 * 768:
                continue
        elif op == "linear":
            c = _lin("", size(1, 32768), size(8, 2048), size(8, 2048), dtype, train,
                     rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.75, rng.random() < 0.5)
            # fp32 products run at a small fraction of the bf16 rate
            if c["rows"] * c["n"] * c["k"] * (1 if dtype == "bf16" else 16) > 32768 * 1536 * 768:
                continue
        else:
            c = _scan("", size(1, 256), size(1, 16384), size(2, 1536), dtype, train,
                      rng.choice(["forward", "reverse", "both"]), rng.random() < 0.4, rng.random() < 0.5)
            if c["direction"] == "both":
                c["d"] += c["d"] % 2
            if c["b"] * c["t"] * c["d"] * (1 if dtype == "bf16" else 2) > 2 * 16384 * 1024:
                continue
        del c["name"]
        return c


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    if own:
        path = os.path.join(os.getcwd(), "rcnn-ocr_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import crnn_hip
        crnn_hip.lib()
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rnd(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        m, n = case["rows"], case["n"]
        # activations of a residual stream: rows of different spread, off centre
        s["x"] = (torch.randn(m, n, generator=g, device=DEV) * (0.5 + torch.rand(m, 1, generator=g, device=DEV))
                  + 0.5 * torch.randn(m, 1, generator=g, device=DEV)).to(dt)
        s["w"] = rnd(n, scale=0.2, shift=1.0, dtype=torch.float32)
        s["b"] = rnd(n, scale=0.2, dtype=torch.float32)
        s["dy"] = rnd(m, n)
        leaves = ("x", "w", "b")
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s["x"] = rnd(m, k)
        s["w"] = rnd(n, k, scale=1.0 / math.sqrt(k))
        s["b"] = rnd(n, scale=0.2) if case["bias"] else None
        s["res"] = rnd(m, n) if case["res"] else None
        s["dy"] = rnd(m, n)
        leaves = ("x", "w", "b", "res")
    else:
        b, t, d = case["b"], case["t"], case["d"]
        # gates biased to remember, as such layers are initialised
        s["f"] = rnd(b, t, d, scale=1.5, shift=1.0)
        s["v"] = rnd(b, t, d)
        s["h0"] = rnd(b, d, dtype=torch.float32) if case["state"] else None
        s["dy"] = rnd(b, t, d)
        s["dhT"] = rnd(b, d, dtype=torch.float32) if case["state"] else None
        s["len"] = None
        if case["ragged"]:
            ln = torch.randint(0, t + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
            ln[0] = t
            if b > 2:
                ln[1], ln[2] = 0, 1
            s["len"] = ln
        leaves = ("f", "v", "h0")
    s["leaves"] = [k for k in leaves if s[k] is not None]
    if case["train"]:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _erf_gelu(z):
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _act(kind, z):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return _erf_gelu(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    return z


def _dact(kind, z):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2 * math.pi))
    sg = torch.sigmoid(z)
    return sg * (1.0 + z * (1.0 - sg))


def _plain_layer_norm(s):
    x = s["x"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * s["w"] + s["b"]).to(s["x"].dtype)
    if not s["case"]["train"]:
        return [y]
    dy = s["dy"].float()
    g = dy * s["w"]
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return [y, dx.to(y.dtype), (dy * xh).sum(0), dy.sum(0)]


def _plain_linear(s):
    c = s["case"]
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if c["bias"]:
        z = z + s["b"].float()
    y = _act(c["act"], z)
    if c["res"]:
        y = y + s["res"].float()
    out = [y.to(dt)]
    if c["train"]:
        dz = s["dy"].float()
        if c["act"] != "none":
            dz = dz * _dact(c["act"], z)
        out += [(dz @ w).to(dt), (dz.t() @ x).to(dt)]
        if c["bias"]:
            out.append(dz.sum(0).to(dt))
        if c["res"]:
            out.append(s["dy"].clone())
    return out


def _doubling(a, b):
    """inclusive scan of h_t = a_t h_{t-1} + b_t over dim 1 (h_{-1} = 0), by doubling: log2 T passes"""
    t, k = a.shape[1], 1
    while k < t:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        if 2 * k < t:
            a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _by_direction(direction, d):
    """(channels, runs backwards) of each part"""
    if direction == "both":
        return [(slice(0, d // 2), False), (slice(d // 2, d), True)]
    return [(slice(0, d), direction == "reverse")]


def _plain_gated_scan(s):
    c = s["case"]
    b, t, d = c["b"], c["t"], c["d"]
    dt = s["f"].dtype
    keep = None
    if s["len"] is not None:   # steps behind a sequence's end hold the state: a = 1, (1 - a) v = 0
        keep = (torch.arange(t, device=DEV)[None, :] < s["len"][:, None])[:, :, None]
    ys, hts, dfs, dvs, dh0s = [], [], [], [], []
    for ch, rev in _by_direction(c["direction"], d):
        turn = (lambda u: u.flip(1)) if rev else (lambda u: u)
        f, v = turn(s["f"][:, :, ch]).float(), turn(s["v"][:, :, ch]).float()
        kp = turn(keep) if keep is not None else None
        a, r = torch.sigmoid(f), torch.sigmoid(-f)
        if kp is not None:
            zero = torch.zeros((), device=DEV)
            a, r, v = torch.where(kp, a, zero + 1.0), torch.where(kp, r, zero), torch.where(kp, v, zero)
        u = r * v
        h0 = s["h0"][:, ch] if s["h0"] is not None else None
        if h0 is not None:
            u = torch.cat([u[:, :1] + a[:, :1] * h0[:, None], u[:, 1:]], 1)
        h = _doubling(a, u)
        y = h if kp is None else torch.where(kp, h, zero)
        ys.append(turn(y).to(dt))
        hts.append(h[:, -1])
        if not c["train"]:
            continue
        dy = turn(s["dy"][:, :, ch]).float()
        if kp is not None:
            dy = torch.where(kp, dy, zero)
        if s["dhT"] is not None:
            dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dhT"][:, None, ch]], 1)
        # G_t = dy_t + a_{t+1} G_{t+1}
        an = torch.cat([torch.zeros_like(a[:, :1]), a.flip(1)[:, :-1]], 1)
        gg = _doubling(an, dy.flip(1)).flip(1)
        hp = torch.cat([h0[:, None] if h0 is not None else torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
        dfs.append(turn(gg * (hp - v) * a * r).to(dt))
        dvs.append(turn(gg * r).to(dt))
        dh0s.append(a[:, 0] * gg[:, 0])
    out = [torch.cat(ys, 2)]
    if c["state"]:
        out.append(torch.cat(hts, 1))
    if c["train"]:
        out += [torch.cat(dfs, 2), torch.cat(dvs, 2)]
        if c["state"]:
            out.append(torch.cat(dh0s, 1))
    return out


def _plain(s):
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "linear": _plain_linear, "gated_scan": _plain_gated_scan}[
            s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------------ the operators
def _forward(s):
    import crnn_hip
    c = s["case"]
    if c["op"] == "layer_norm":
        return (crnn_hip.layer_norm(s["x"], s["w"], s["b"], EPS),)
    if c["op"] == "linear":
        return (crnn_hip.linear(s["x"], s["w"], s["b"], activation=c["act"], residual=s["res"]),)
    out = crnn_hip.gated_scan(s["f"], s["v"], h0=s["h0"], lengths=s["len"], direction=c["direction"],
                              return_state=c["state"])
    return out if c["state"] else (out,)


def run(state):
    if not own:
        return _plain(state)
    if not state["case"]["train"]:
        with torch.no_grad():
            return list(_forward(state))
    out = _forward(state)
    up = [state["dy"]] + ([state["dhT"]] if len(out) > 1 else [])
    grads = torch.autograd.grad(out, [state[k] for k in state["leaves"]], up)
    return [o.detach() for o in out] + list(grads)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "layer_norm":
        m, n = case["rows"], case["n"]
        x = m * n * e
        if case["train"]:   # x, dy, weight, bias in; y, dx, dweight, dbias out
            return {"bytes": 4 * x + 4 * n * 4, "flops": 20 * m * n}
        return {"bytes": 2 * x + 2 * n * 4, "flops": 8 * m * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        one, bias, res = m * n * e, n * e * case["bias"], m * n * e * case["res"]
        if case["train"]:   # x, w, dy (+ bias, residual) in; y, dx, dw (+ dbias, dresidual) out
            return {"bytes": 2 * m * k * e + 2 * n * k * e + 2 * one + 2 * bias + 2 * res, "flops": 6 * m * n * k}
        return {"bytes": m * k * e + n * k * e + one + bias + res, "flops": 2 * m * n * k}
    b, t, d = case["b"], case["t"], case["d"]
    x, st = b * t * d * e, b * d * 4 * case["state"]
    if case["train"]:   # f, v, dy (+ h0, dhT) in; y, df, dv (+ hT, dh0) out
        return {"bytes": 6 * x + 4 * st, "flops": 25 * b * t * d}
    return {"bytes": 3 * x + 2 * st, "flops": 8 * b * t * d}


# ------------------------------------------------------------------------------------------------ the definitions in fp64
def _exact_layer_norm(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    n = x.shape[-1]
    mean = x.sum(1) / n
    var = ((x - mean[:, None]) ** 2).sum(1) / n
    sd = (var + EPS).sqrt()
    xh = (x - mean[:, None]) / sd[:, None]
    out = [torch.addcmul(b, xh, w)]
    if s["case"]["train"]:
        dy = s["dy"].double()
        dxh = dy * w
        # d xhat_j / d x_i = (delta_ij - 1/n - xhat_i xhat_j / n) / sd
        c1, c2 = dxh.sum(1), (dxh * xh).sum(1)
        out += [(n * dxh - c1[:, None] - c2[:, None] * xh) / (n * sd[:, None]), (xh * dy).sum(0), dy.sum(0)]
    return out


def _exact_linear(s):
    c = s["case"]
    x, w = s["x"].double(), s["w"].double()
    z = torch.mm(x, w.t().contiguous())
    if s["b"] is not None:
        z += s["b"].double()
    cdf = torch.special.ndtr(z)
    lg = torch.special.expit(z)
    y, dz = {"none": (z, None), "relu": (z.clamp(min=0), z.sign().clamp(min=0)),
             "gelu": (z * cdf, cdf + z * (z * z / -2).exp() / (2 * math.pi) ** 0.5),
             "silu": (z * lg, lg + z * lg * (1 - lg))}[c["act"]]
    if s["res"] is not None:
        y = y + s["res"].double()
    out = [y]
    if c["train"]:
        dy = s["dy"].double()
        g = dy if dz is None else dz * dy
        out += [torch.mm(g, w), torch.mm(g.t().contiguous(), x)]
        if s["b"] is not None:
            out.append(g.sum(0))
        if s["res"] is not None:
            out.append(dy)
    return out


def _exact_gated_scan(s):
    """step by step, as the recurrence is written; the gradient by walking the steps back"""
    c = s["case"]
    b, t, d = c["b"], c["t"], c["d"]
    f, v = s["f"].double().transpose(0, 1).contiguous(), s["v"].double().transpose(0, 1).contiguous()
    a, r = torch.special.expit(f), torch.special.expit(-f)
    on = None
    if s["len"] is not None:
        on = (torch.arange(t, device=DEV)[:, None] < s["len"][None, :])[:, :, None].expand(t, b, d)
        a, r, v = a.masked_fill(~on, 1), r.masked_fill(~on, 0), v.masked_fill(~on, 0)
    u = r * v
    h = torch.empty_like(u)
    hp = torch.empty_like(u)
    start = s["h0"].double() if s["h0"] is not None else torch.zeros(b, d, dtype=torch.float64, device=DEV)
    dy = s["dy"].double().transpose(0, 1).contiguous()
    if on is not None:
        dy = dy.masked_fill(~on, 0)
    gg, first = torch.empty_like(u), torch.empty_like(start)
    last = torch.empty_like(start)
    half = d // 2
    for lo, hi, steps in {"forward": [(0, d, 1)], "reverse": [(0, d, -1)],
                          "both": [(0, half, 1), (half, d, -1)]}[c["direction"]]:
        order = range(t)[::steps]
        cur = start[:, lo:hi]
        for i in order:
            hp[i, :, lo:hi] = cur
            cur = torch.addcmul(u[i, :, lo:hi], a[i, :, lo:hi], cur, out=h[i, :, lo:hi])
        last[:, lo:hi] = cur
        if c["train"]:
            carry = s["dhT"][:, lo:hi].double() if s["dhT"] is not None else torch.zeros_like(start[:, lo:hi])
            for i in reversed(order):
                torch.add(dy[i, :, lo:hi], carry, out=gg[i, :, lo:hi])
                carry = a[i, :, lo:hi] * gg[i, :, lo:hi]
            first[:, lo:hi] = carry
    y = h if on is None else h.masked_fill(~on, 0)
    out = [y.transpose(0, 1).contiguous()]
    if c["state"]:
        out.append(last)
    if c["train"]:
        out += [(gg * (hp - v) * a * r).transpose(0, 1).contiguous(), (gg * r).transpose(0, 1).contiguous()]
        if c["state"]:
            out.append(first)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"layer_norm": _exact_layer_norm, "linear": _exact_linear, "gated_scan": _exact_gated_scan}[
            case["op"]](s)
