"""The sequence operators (crnn_hip.layer_norm, linear, gated_scan) against plain fp64 implementations, element by element.

Tolerances are bounds, not fits. U = 2^-24 is half a step of fp32, ET half a step of the result's type (bf16 2^-8, fp32 U);
each reference returns, beside a value, a bound on what rounding may do to it: a rounded result ET |y|; a sum of n fp32
terms (n + a small constant) U times the sum of their magnitudes; and first-order propagation from there, with the
constants K below covering the handful of elementary operations (exp, reciprocal, multiply) of each formula."""
import math

import pytest
import torch

import crnn_hip
from crnn_hip import _lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
ET = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
TYPES = [torch.float32, torch.bfloat16]
TINY = 1e-37   # results below the smallest normals may be flushed


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)


def within(name, got, ref, bound):
    got = got.detach().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    if got.numel() == 0:
        return
    over = ((got - ref).abs() / (bound + TINY)).max()
    assert float(over) <= 1.0, f"{name}: {float(over):.3g} times its bound"


# ------------------------------------------------------------------------------------------------ layer norm
def ln_ref(x, w, b, dy, eps, dt):
    x, dy = x.double(), dy.double()
    m, n = x.shape
    w = w.double() if w is not None else torch.ones(n, dtype=torch.float64, device=DEV)
    b = b.double() if b is not None else torch.zeros(n, dtype=torch.float64, device=DEV)
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rs = 1 / ((xc * xc).mean(1, keepdim=True) + eps).sqrt()
    xh = xc * rs
    y = xh * w + b
    # xhat: the mean is good to a few U max|x| and rstd to a few U plus what that error of the mean does
    R = 1 + rs * x.abs().max(1, keepdim=True).values
    K = 32 * U
    exh = K * (xh.abs() + R)
    ey = ET[dt] * y.abs() + exh * w.abs() + K * (y.abs() + b.abs())
    g = dy * w
    s1, s2, a1, a2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True), g.abs().mean(1, keepdim=True), \
        (g * xh).abs().mean(1, keepdim=True)
    dx = rs * (g - s1 - xh * s2)
    edx = ET[dt] * dx.abs() + rs * K * (g.abs() + a1 + xh.abs() * a2 + R * (s2.abs() + xh.abs() * a1))
    n_add = (m / 512 + 64) * U
    dw, db = (dy * xh).sum(0), dy.sum(0)
    edw = (dy.abs() * exh).sum(0) + n_add * (dy * xh).abs().sum(0)
    edb = n_add * dy.abs().sum(0)
    return (y, ey), (dx, edx), (dw, edw), (db, edb)


LN_SIZES = [(1, 1), (3, 7), (31, 8), (7, 65), (2003, 100), (1001, 128), (15, 129), (4099, 250), (3, 256), (2, 257),
            (1, 512), (5, 513), (17, 64), (1000, 512), (301, 768), (130, 1021), (9, 1024), (7, 1025), (6, 2048), (33, 2049),
            (5, 4096), (3, 4097), (4, 8192), (3, 10007), (2, 16384), (3, 16385), (2, 40001), (6000, 33)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n", LN_SIZES)
def test_layer_norm(m, n, dt):
    g = gen(m * 1000003 + n)
    x = (randn(g, m, n) * (0.2 + randn(g, m, 1).abs()) + 3 * randn(g, m, 1)).to(dt)
    w, b, dy = randn(g, n, shift=1.0, scale=0.3), randn(g, n), randn(g, m, n, dtype=dt)
    for ww, bb in ((w, b), (None, None), (w, None), (None, b)):
        leaves = [t.clone().requires_grad_(True) for t in (x, ww, bb) if t is not None]
        lx = leaves[0]
        lw = leaves[1] if ww is not None else None
        lb = leaves[-1] if bb is not None else None
        y = crnn_hip.layer_norm(lx, lw, lb, 1e-5)
        assert y.dtype == dt
        grads = list(torch.autograd.grad(y, leaves, dy))
        refs = ln_ref(x, ww, bb, dy, 1e-5, dt)
        within("y", y, *refs[0])
        within("dx", grads.pop(0), *refs[1])
        if ww is not None:
            assert grads[0].dtype == torch.float32
            within("dw", grads.pop(0), *refs[2])
        if bb is not None:
            within("db", grads.pop(0), *refs[3])
        with torch.no_grad():
            assert torch.equal(crnn_hip.layer_norm(x, ww, bb, 1e-5), y)   # inference: the same numbers


@pytest.mark.parametrize("dt", TYPES)
def test_layer_norm_layouts(dt):
    """leading axes, strided and unaligned rows, rows that are not rows (copied), no rows, constant and far-off rows"""
    g = gen(5)
    n = 70
    w, b = randn(g, n, shift=1.0), randn(g, n)
    base = randn(g, 6, 5, 200, dtype=dt)
    for x in (base[..., :n], base[..., 3:3 + n], base[:, :, 1:2 * n + 1:2], base.transpose(0, 1)[..., 7:7 + n], base[0, 0, :n],
              base[:1, :1, :n].expand(4, 3, n)):
        ref = ln_ref(x.reshape(-1, n), w, b, torch.zeros_like(x.reshape(-1, n)), 1e-5, dt)[0]
        y = crnn_hip.layer_norm(x, w, b)
        assert y.shape == x.shape
        within("y", y.reshape(-1, n), *ref)
    x = torch.empty(0, 4, n, device=DEV, dtype=dt, requires_grad=True)
    lw = w.clone().requires_grad_(True)
    y = crnn_hip.layer_norm(x, lw, b)
    assert y.shape == (0, 4, n)
    gx, gw = torch.autograd.grad(y, (x, lw), torch.empty_like(y))
    assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(gw))
    c = torch.full((3, n), 100.0, device=DEV, dtype=dt)     # variance 0: y = b
    assert torch.equal(crnn_hip.layer_norm(c, w, b), b.to(dt).expand(3, n))
    far = (randn(g, 4, n) + 3000.0).to(dt)                   # bf16 keeps few steps there; fp32 keeps the variance
    within("far", crnn_hip.layer_norm(far, w, b), *ln_ref(far, w, b, torch.zeros_like(far), 1e-5, dt)[0])


@pytest.mark.parametrize("n", [5, 60, 100, 256])
def test_layer_norm_rows_of_a_wave_do_not_mix(n):
    """narrow rows share a wave: a NaN or infinity stays in its own, forward and backward"""
    g = gen(n)
    x, dy = randn(g, 37, n), randn(g, 37, n)
    keep = [i for i in range(37) if i not in (3, 7, 36)]

    def run(x):
        lx = x.clone().requires_grad_(True)
        y = crnn_hip.layer_norm(lx)
        return y.detach(), torch.autograd.grad(y, lx, dy)[0]
    x2 = x.clone()
    x2[3, n - 1], x2[7, 1], x2[36, 0] = float("nan"), float("inf"), float("-inf")
    for a, b in zip(run(x), run(x2)):
        assert torch.equal(a[keep], b[keep]) and torch.isnan(b[[3, 7, 36]]).all()


def test_layer_norm_rows_do_not_mix():
    """a NaN or infinite row stays its own; the strided output of a wider buffer's neighbours is not touched"""
    g = gen(6)
    x = randn(g, 9, 512)
    y = crnn_hip.layer_norm(x)
    x2 = x.clone()
    x2[3, 5], x2[7, 1] = float("nan"), float("inf")
    y2 = crnn_hip.layer_norm(x2)
    keep = [i for i in range(9) if i not in (3, 7)]
    assert torch.equal(y2[keep], y[keep]) and torch.isnan(y2[[3, 7]]).all()
    buf = torch.full((9, 600), 7.0, device=DEV)
    L.call("crnn_layernorm_fwd", 0, x.data_ptr(), 512, None, None, buf.data_ptr(), 600, None, None, 9, 512, 1e-5, L.stream_ptr())
    assert torch.equal(buf[:, :512], y) and (buf[:, 512:] == 7.0).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [40, 96, 200, 1500, 20000])
def test_layer_norm_residual_gradient_and_accumulation(n, dt):
    """the C entry's dres (added before dx's one rounding, in place too) and accumulate"""
    g = gen(n)
    m = 37
    x, dy, dres = randn(g, m, n, dtype=dt), randn(g, m, n, dtype=dt), randn(g, m, n, dtype=dt)
    w = randn(g, n, shift=1.0)
    code, s = L.dtype_code(dt), L.stream_ptr()
    y, mean, rstd = torch.empty_like(x), torch.empty(m, device=DEV), torch.empty(m, device=DEV)
    L.call("crnn_layernorm_fwd", code, x.data_ptr(), n, w.data_ptr(), None, y.data_ptr(), n, mean.data_ptr(), rstd.data_ptr(), m, n,
           1e-5, s)
    need = L.lib().crnn_layernorm_bwd_workspace(code, m, n)
    ws = torch.empty(need // 4, device=DEV)
    dw, db = torch.full((n,), 2.0, device=DEV), torch.full((n,), 3.0, device=DEV)
    dx = dres.clone()
    L.call("crnn_layernorm_bwd", code, dy.data_ptr(), n, x.data_ptr(), n, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
           dx.data_ptr(), n, dx.data_ptr(), n, dw.data_ptr(), db.data_ptr(), 1, ws.data_ptr(), need, m, n, s)
    _, (rx, ex), (rw, ew), (rb, eb) = ln_ref(x, w, None, dy, 1e-5, dt)
    rx2 = rx + dres.double()
    within("dx + dres", dx, rx2, ex + ET[dt] * rx2.abs() + 2 * U * (rx.abs() + dres.double().abs()))
    within("dw +=", dw, rw + 2.0, ew + 2 * U * (rw.abs() + 2))
    within("db +=", db, rb + 3.0, eb + 2 * U * (rb.abs() + 3))


# ------------------------------------------------------------------------------------------------ linear
# act, act', and a bound on |act''| (how far a rounded pre-activation moves act')
ACTS = {"none": (lambda z: z, lambda z: torch.ones_like(z), 0.0),
        "relu": (lambda z: z.clamp(min=0), lambda z: (z > 0).double(), 0.0),
        "gelu": (lambda z: z * torch.special.ndtr(z),
                 lambda z: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8),
        "silu": (lambda z: z * torch.sigmoid(z), lambda z: torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z))), 0.5)}
APPROX = {torch.bfloat16: 1e-5, torch.float32: 16 * U}   # the activation functions themselves (fast forms 4e-6 and a few U)


def linear_ref(x, w, b, res, dy, kind, dt):
    fn, dfn, curve = ACTS[kind]
    x, w, dy = x.double(), w.double(), dy.double()
    m, k = x.shape
    n = w.shape[0]
    z = x @ w.t().contiguous()
    S = x.abs() @ w.abs().t().contiguous()
    if b is not None:
        z, S = z + b.double(), S + b.double().abs()
    ez = (k / 4 + 16) * U * S
    y = fn(z)
    ey = 1.2 * ez + APPROX[dt] * (1 + z.abs()) * (kind != "none") + 4 * U * z.abs()
    if res is not None:
        y = y + res.double()
        ey = ey + 2 * U * (res.double().abs() + y.abs())
    ey = ey + ET[dt] * y.abs()
    d = dfn(z)
    dz = dy * d
    edz = dy.abs() * (curve * (ET[dt] * z.abs() + ez) + APPROX[dt] * (1 + z.abs()) * (kind != "none")) + 2 * U * dz.abs()
    if kind == "relu":
        edz = edz + dy.abs() * (z.abs() <= ez)   # a sum next to 0 may fall on the other side
    edb = edz.sum(0) + (m / 4 + 16) * U * dz.abs().sum(0)
    edz = edz + ET[dt] * dz.abs() * (kind != "none")   # rounded for the products
    dx, dw, db = dz @ w, dz.t().contiguous() @ x, dz.sum(0)
    edx = edz @ w.abs() + (n / 4 + 16) * U * (dz.abs() @ w.abs()) + ET[dt] * dx.abs()
    edw = edz.t().contiguous() @ x.abs() + (m / 4 + 16) * U * (dz.abs().t().contiguous() @ x.abs()) + ET[dt] * dw.abs()
    return (y, ey), (dx, edx), (dw, edw), (db, edb)


LIN_SIZES = [(1, 1, 1), (1, 512, 1024), (3, 9, 5), (16, 512, 1024), (17, 40, 24), (33, 509, 130), (64, 256, 64), (65, 256, 257),
             (130, 127, 129), (257, 64, 8), (300, 1000, 513), (1027, 509, 1021), (2048, 512, 1024), (6150, 256, 520), (5000, 8, 2000)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", LIN_SIZES)
def test_linear(m, k, n, dt):
    g = gen(m * 7 + k * 11 + n)
    x, w = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=1 / math.sqrt(k))
    b, res, dy = randn(g, n, dtype=dt), randn(g, m, n, dtype=dt), randn(g, m, n, dtype=dt)
    for kind, bias, r in (("none", None, None), ("gelu", b, None), ("silu", b.float(), res), ("relu", b, res), ("none", b.float(), res)):
        leaves = [t.clone().requires_grad_(True) if t is not None else None for t in (x, w, bias, r)]
        y = crnn_hip.linear(leaves[0], leaves[1], leaves[2], activation=kind, residual=leaves[3])
        assert y.dtype == dt
        has = [t for t in leaves if t is not None]
        grads = list(torch.autograd.grad(y, has, dy))
        (ry, ey), (rx, ex), (rw, ew), (rb, eb) = linear_ref(x, w, bias, r, dy, kind, dt)
        within(f"{kind} y", y, ry, ey)
        within(f"{kind} dx", grads[0], rx, ex)
        within(f"{kind} dw", grads[1], rw, ew)
        if bias is not None:
            assert grads[2].dtype == bias.dtype
            within(f"{kind} db", grads[2], rb, eb + ET[bias.dtype] * rb.abs())
        if r is not None:
            assert torch.equal(grads[-1], dy)
        with torch.no_grad():
            assert torch.equal(crnn_hip.linear(x, w, bias, activation=kind, residual=r), y)


@pytest.mark.parametrize("dt", TYPES)
def test_linear_layouts_and_subsets(dt):
    """leading axes, strided / unaligned / transposed operands, no rows, gradients of a subset, an expanded upstream gradient"""
    g = gen(11)
    k, n = 72, 48
    base, wb = randn(g, 4, 9, 200, dtype=dt), randn(g, 100, 200, dtype=dt, scale=0.1)
    res = randn(g, 4, 9, 100, dtype=dt)
    dy = randn(g, 36, n, dtype=dt)
    for x in (base[..., :k], base[..., 8:8 + k], base[..., 3:3 + k], base[:, :, 1:2 * k:2], base[0, :, :k], base[0, 0, 5:5 + k]):
        for w in (wb[:n, :k], wb[1:n + 1, 5:5 + k], wb.t()[:n, :k]):
            r = res[..., 1:1 + n] if x.dim() == 3 else None
            y = crnn_hip.linear(x, w, None, activation="gelu", residual=r)
            assert y.shape == x.shape[:-1] + (n,)
            x2 = x.reshape(-1, k)
            ref = linear_ref(x2, w, None, r.reshape(-1, n) if r is not None else None, dy[:x2.shape[0]], "gelu", dt)[0]
            within("y", y.reshape(-1, n), *ref)
    x, w = base[..., 3:3 + k].detach(), wb[:n, :k].detach()
    x2 = x.reshape(-1, k)
    one = torch.ones((), device=DEV, dtype=dt).expand(4, 9, n)
    refs = linear_ref(x2, w, None, None, one.reshape(-1, n), "silu", dt)
    for which in ("x", "w"):
        lx, lw = x.clone().requires_grad_(which == "x"), w.clone().requires_grad_(which == "w")
        (gr,) = torch.autograd.grad(crnn_hip.linear(lx, lw, activation="silu"), [lx if which == "x" else lw], one)
        within("d" + which, gr.reshape(-1, k), *refs[1 if which == "x" else 2])
    lx, lw, lb = (t.clone().requires_grad_(True) for t in (x[:0], w, wb[0, :n]))
    y = crnn_hip.linear(lx, lw, lb, activation="relu")
    assert y.shape == (0, 9, n)
    gx, gw, gb = torch.autograd.grad(y, (lx, lw, lb), torch.empty_like(y))
    assert gx.shape == lx.shape and not gw.any() and not gb.any()


def test_linear_c_entry_accumulates_and_keeps_neighbours():
    g = gen(12)
    m, k, n = 300, 64, 56
    x, w, dy = (randn(g, *s, dtype=torch.bfloat16) for s in ((m, k), (n, k), (m, n)))
    s = L.stream_ptr()
    buf = torch.full((m, 80), 7.0, device=DEV, dtype=torch.bfloat16)
    L.call("crnn_linear_fwd", 1, x.data_ptr(), k, w.data_ptr(), k, None, 0, 0, None, 0, buf.data_ptr(), 80, None, 0, None, 0, m, n, k, s)
    assert torch.equal(buf[:, :n], crnn_hip.linear(x, w)) and (buf[:, n:] == 7.0).all()
    dw, db = torch.full((n, k), 2.0, device=DEV), torch.full((n,), 3.0, device=DEV)
    dx = torch.full((m, 100), 7.0, device=DEV, dtype=torch.bfloat16)
    need = L.lib().crnn_linear_bwd_workspace(1, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, 0, 1, 1, 1, m, n, k)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    L.call("crnn_linear_bwd", 1, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, None, 0, 0, dx.data_ptr(), 100, dw.data_ptr(), 1,
           db.data_ptr(), 1, 1, ws.data_ptr(), need, m, n, k, s)
    _, (rx, ex), (rw, ew), (rb, eb) = linear_ref(x, w, None, None, dy, "none", torch.bfloat16)
    within("dx", dx[:, :k], rx, ex)
    assert (dx[:, k:] == 7.0).all()
    within("dw +=", dw, rw + 2, ew + 2 * U * (rw.abs() + 2))
    within("db +=", db, rb + 3, eb + 2 * U * (rb.abs() + 3))


# ------------------------------------------------------------------------------------------------ gated scan
def scan_ref(f, v, h0, lengths, dy, dhT, direction, dt):
    """the recurrence walked step by step in fp64, and beside it how far rounding may have moved state and gradient: each step
    adds a few roundings of its terms and what the gate's relative error ((4 + |f|) U through exp) does to them; the same
    bound covers the composed pieces, whose products are of the same gates"""
    f, v, dy = f.double(), v.double(), dy.double()
    B, T, D = f.shape
    K = 8 * U
    dev = f.device
    lens = lengths.clamp(0, T).tolist() if lengths is not None else [T] * B
    a, r = torch.sigmoid(f), torch.sigmoid(-f)
    y, hp, ehp, G, eG = (torch.zeros_like(f) for _ in range(5))
    ey = torch.zeros_like(f)
    hT = h0.double().clone() if h0 is not None else torch.zeros(B, D, dtype=torch.float64, device=dev)
    d0 = dhT.double().clone() if dhT is not None else torch.zeros_like(hT)
    ehT, ed0 = torch.zeros_like(hT), torch.zeros_like(hT)
    half = {"forward": D, "reverse": 0, "both": D // 2}[direction]
    # all samples and channels walk together in "walking order"; t(u) per sample and direction
    for ch, rev in ((slice(0, half), False), (slice(half, D), True)):
        if ch.stop - ch.start == 0:
            continue
        idx = torch.zeros(B, T, dtype=torch.long, device=dev)
        on = torch.zeros(B, T, 1, dtype=torch.bool, device=dev)
        for b, n in enumerate(lens):
            u = torch.arange(T, device=dev)
            idx[b] = torch.where(u < n, (n - 1 - u) if rev else u, u)
            on[b, :n] = True
        ix = idx[:, :, None].expand(B, T, ch.stop - ch.start)
        A, Rr, V, Fm, DY = (q[:, :, ch].gather(1, ix) for q in (a, r, v, f, dy))
        A, Rr = torch.where(on, A, torch.ones_like(A)), torch.where(on, Rr, torch.zeros_like(Rr))
        V, DY, gerr = (torch.where(on, q, torch.zeros_like(q)) for q in (V, DY, 4 + Fm.abs()))
        h, e = hT[:, ch].clone(), torch.zeros_like(hT[:, ch])
        hs, es, hps, ehps = [], [], [], []
        for u in range(T):
            hps.append(h)
            ehps.append(e)
            e = A[:, u] * e + K * ((A[:, u] * h).abs() + (Rr[:, u] * V[:, u]).abs() + A[:, u] * Rr[:, u] * (h.abs() + V[:, u].abs()) * gerr[:, u])
            h = A[:, u] * h + Rr[:, u] * V[:, u]
            hs.append(h)
            es.append(e)
        hT[:, ch], ehT[:, ch] = h, e
        c, ec = d0[:, ch].clone(), torch.zeros_like(h)
        gs, egs = [None] * T, [None] * T
        for u in reversed(range(T)):
            gg = DY[:, u] + c
            eg = ec + K * (DY[:, u].abs() + c.abs())
            gs[u], egs[u] = gg, eg
            c = A[:, u] * gg
            ec = A[:, u] * eg + K * (c.abs() + A[:, u] * Rr[:, u] * gg.abs() * gerr[:, u])
        d0[:, ch], ed0[:, ch] = c, ec
        st = lambda q: torch.stack(q, 1) if q else torch.zeros(B, 0, ch.stop - ch.start, dtype=torch.float64, device=dev)  # noqa: E731
        zero = torch.zeros((), dtype=torch.float64, device=dev)
        for dst, src in ((y, hs), (ey, es), (hp, hps), (ehp, ehps), (G, gs), (eG, egs)):
            dst[:, :, ch] = torch.zeros_like(dst[:, :, ch]).scatter(1, ix, torch.where(on, st(src), zero))
    mask = torch.zeros(B, T, 1, dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        mask[b, :n] = True
    zero = torch.zeros((), dtype=torch.float64, device=dev)
    vv, ge = torch.where(mask, v, zero), 4 + torch.where(mask, f, zero).abs()
    rr, aa = torch.where(mask, r, zero), torch.where(mask, a, zero)
    df, dv = G * (hp - vv) * aa * rr, G * rr
    edv = eG * rr + K * dv.abs() * ge + ET[dt] * dv.abs()
    edf = aa * rr * (eG * (hp - vv).abs() + G.abs() * ehp + K * G.abs() * (hp.abs() + vv.abs())) + 2 * K * df.abs() * ge + ET[dt] * df.abs()
    return (y, ey + ET[dt] * y.abs()), (hT, ehT), (df, edf), (dv, edv), (d0, ed0)


def scan_check(f, v, h0, lengths, direction, g, dt, state=True):
    B, T, D = f.shape
    dy = randn(g, B, T, D, dtype=dt)
    dhT = randn(g, B, D) if state else None
    lf, lv = f.detach().requires_grad_(True), v.detach().requires_grad_(True)
    lh = h0.clone().requires_grad_(True) if h0 is not None else None
    out = crnn_hip.gated_scan(lf, lv, h0=lh, lengths=lengths, direction=direction, return_state=state)
    outs = out if state else (out,)
    leaves = [t for t in (lf, lv, lh) if t is not None]
    grads = torch.autograd.grad(outs, leaves, [dy] + ([dhT] if state else []))
    ry, rh, rf, rv, r0 = scan_ref(f, v, h0, lengths, dy, dhT, direction, dt)
    within("y", outs[0], *ry)
    if state:
        within("hT", outs[1], *rh)
    within("df", grads[0], *rf)
    within("dv", grads[1], *rv)
    if h0 is not None:
        within("dh0", grads[2], *r0)
    if lengths is not None:
        for b, n in enumerate(lengths.clamp(0, T).tolist()):
            assert not outs[0][b, n:].any() and not grads[0][b, n:].any() and not grads[1][b, n:].any()
    with torch.no_grad():
        again = crnn_hip.gated_scan(f, v, h0=h0, lengths=lengths, direction=direction, return_state=state)
        assert torch.equal(again[0] if state else again, outs[0])
        if state:
            assert torch.equal(again[1], outs[1])


SCAN_SIZES = [(1, 1, 2), (3, 1, 130), (2, 2, 6), (5, 7, 128), (4, 8, 130), (3, 9, 62), (2, 16, 256), (3, 17, 258), (7, 33, 64),
              (256, 32, 64), (4, 64, 130), (1, 129, 1024), (2, 257, 66), (1, 700, 2), (1, 4097, 130), (2, 1500, 258), (40, 300, 300)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("direction", ["forward", "reverse", "both"])
@pytest.mark.parametrize("b,t,d", SCAN_SIZES)
def test_gated_scan(b, t, d, direction, dt):
    g = gen(b * 31 + t * 17 + d)
    d -= d % 4 // 2 if direction != "both" else 0   # odd half-widths too
    if direction != "both" and d > 2:
        d -= 1
    f, v, h0 = randn(g, b, t, d, dtype=dt, scale=2.0, shift=1.0), randn(g, b, t, d, dtype=dt), randn(g, b, d)
    scan_check(f, v, h0, None, direction, g, dt)
    scan_check(f, v, None, None, direction, g, dt, state=False)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("direction", ["forward", "reverse", "both"])
@pytest.mark.parametrize("b,t,d", [(5, 8, 66), (6, 37, 130), (5, 300, 34), (2, 2500, 66), (3, 2100, 10)])
def test_gated_scan_lengths(b, t, d, direction, dt):
    """empty, one-step, ragged and out-of-range lengths; what lies behind a length (NaN, infinities) is not read"""
    g = gen(b + t + d)
    f, v, h0 = randn(g, b, t, d, dtype=dt, scale=2.0), randn(g, b, t, d, dtype=dt), randn(g, b, d)
    lens = torch.randint(0, t + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    lens[0], lens[1] = 0, 1
    if b > 2:
        lens[2] = t + 5   # clamped
    if b > 4:
        lens[3], lens[4] = -3, t // 2 + 1
    for i, n in enumerate(lens.clamp(0, t).tolist()):
        f[i, n:], v[i, n:] = float("nan"), float("inf")
    scan_check(f, v, h0, lens, direction, g, dt)
    same = crnn_hip.gated_scan(f, v, h0=h0, lengths=lens.long() + (lens.long() >= t).long() * (1 << 33), direction=direction)
    assert torch.equal(same, crnn_hip.gated_scan(f, v, h0=h0, lengths=lens, direction=direction))


@pytest.mark.parametrize("dt", TYPES)
def test_gated_scan_views_and_gates(dt):
    """halves of one projection, time-major and unaligned views; saturated and infinite gate logits; T = 0 and B = 0"""
    g = gen(21)
    B, T, H = 3, 45, 64
    proj = randn(g, B, T, 4 * H + 1, dtype=dt)
    scan_check(proj[..., : 2 * H], proj[..., 2 * H: 4 * H], None, None, "both", g, dt)
    scan_check(proj[..., 1: 2 * H + 1], proj[..., 2 * H + 1:], randn(g, B, 2 * H), None, "both", g, dt)
    tm = randn(g, T, B, H, dtype=dt).transpose(0, 1)
    scan_check(tm, proj[..., :H], None, torch.tensor([45, 9, 0], device=DEV), "reverse", g, dt)
    scan_check(randn(g, B, H, T, dtype=dt).transpose(1, 2), proj[..., :H], None, None, "forward", g, dt)
    f = randn(g, B, T, H, dtype=dt, scale=60.0)   # mostly saturated: copies and resets
    scan_check(f, proj[..., :H], randn(g, B, H), None, "forward", g, dt)
    f = randn(g, B, T, H, dtype=dt)
    f[:, 10:20], f[:, 30:32] = float("inf"), float("-inf")   # hold, then take the new value
    h0 = randn(g, B, H)
    y, hT = crnn_hip.gated_scan(f, proj[..., :H], h0=h0, return_state=True)
    assert torch.equal(y[:, 30:32], proj[:, 30:32, :H])
    # Held steps keep the state, but a state that enters a wave's 8 steps comes through their composed (A, H): A a product of
    # 8 gates (8 U), H a sum of 8 products (16 U max|v|), one multiply-add (2 U): a held stretch may differ by 26 U (|h| + |v|)
    # <= 64 U max(|h0|, |v|) where it crosses from one such piece into the next (once here), and by a step of the type where
    # that falls on two sides of a rounding border
    top = float(torch.maximum(proj.abs().max().float(), h0.abs().max()))
    held = y[:, 9:10].double().expand(B, 10, H)
    within("held", y[:, 10:20], held, 64 * U * top + 2 * ET[dt] * held.abs())
    for shape in ((2, 0, 6), (0, 4, 6), (2, 4, 0)):
        e = torch.zeros(shape, device=DEV, dtype=dt, requires_grad=True)
        h = randn(g, shape[0], shape[2]).requires_grad_(True)
        y, hT = crnn_hip.gated_scan(e, e, h0=h, return_state=True)
        gh, = torch.autograd.grad(hT, h, 2 * torch.ones_like(hT))
        assert y.shape == e.shape
        if shape[1] == 0:
            assert torch.equal(hT, h) and (gh == 2).all()


def test_gated_scan_state_only_and_value_only():
    """the gradient through the final state alone, and through y alone when a state was returned"""
    g = gen(23)
    f, v, h0 = randn(g, 3, 40, 66), randn(g, 3, 40, 66), randn(g, 3, 66)
    for use in ("state", "value"):
        leaves = [t.clone().requires_grad_(True) for t in (f, v, h0)]
        y, hT = crnn_hip.gated_scan(leaves[0], leaves[1], h0=leaves[2], return_state=True)
        dy, dhT = randn(g, 3, 40, 66), randn(g, 3, 66)
        grads = torch.autograd.grad(hT if use == "state" else y, leaves, dhT if use == "state" else dy)
        refs = scan_ref(f, v, h0, None, torch.zeros_like(dy) if use == "state" else dy, dhT if use == "state" else None, "forward",
                        torch.float32)
        for name, got, ref in zip(("df", "dv", "dh0"), grads, refs[2:]):
            within(name, got, *ref)


@pytest.mark.parametrize("dt", TYPES)
def test_gated_scan_continues(dt):
    """a sequence in stretches, and step by step in place, equals the whole one to the rounding of the state's composition"""
    g = gen(22)
    B, T, D = 4, 70, 130
    f, v, h0 = randn(g, B, T, D, dtype=dt, shift=1.0), randn(g, B, T, D, dtype=dt), randn(g, B, D)
    ry, rh, *_ = scan_ref(f, v, h0, None, torch.zeros_like(f), None, "forward", dt)
    parts, h = [], h0
    for a, b in ((0, 1), (1, 30), (30, 31), (31, 70)):
        y, h = crnn_hip.gated_scan(f[:, a:b], v[:, a:b], h0=h, return_state=True)
        parts.append(y)
    within("stretches y", torch.cat(parts, 1), *ry)
    within("stretches hT", h, *rh)
    state, outs = h0.clone(), []
    for t in range(T):
        y, s2 = crnn_hip.gated_scan_step(f[:, t], v[:, t], state, out_state=state)
        assert s2.data_ptr() == state.data_ptr()
        outs.append(y)
    within("steps y", torch.stack(outs, 1), *ry)
    within("steps hT", state, *rh)
    y, new = crnn_hip.gated_scan_step(f[:, 0], v[:, 0], h0)
    assert new.data_ptr() != h0.data_ptr() and torch.equal(y, outs[0])


# ------------------------------------------------------------------------------------------------ all three
def layer(x, p):
    """the run of an encoder layer: norm -> projection -> scan -> projection + residual, norm -> gelu -> projection + residual"""
    h = x.shape[-1]
    u = crnn_hip.linear(crnn_hip.layer_norm(x, p["n1w"], p["n1b"]), p["wi"], p["bi"])
    y = crnn_hip.gated_scan(u[..., : 2 * h], u[..., 2 * h:], direction="both")
    x = crnn_hip.linear(y, p["wo"], p["bo"], residual=x)
    u = crnn_hip.linear(crnn_hip.layer_norm(x, p["n2w"], p["n2b"]), p["w1"], p["b1"], activation="gelu")
    return crnn_hip.linear(u, p["w2"], p["b2"], residual=x)


def layer_params(g, h, dt):
    p = dict(wi=randn(g, 4 * h, h, scale=1 / math.sqrt(h)), bi=randn(g, 4 * h, scale=0.1), wo=randn(g, h, 2 * h, scale=0.5 / math.sqrt(h)),
             bo=randn(g, h, scale=0.1), w1=randn(g, 2 * h, h, scale=1 / math.sqrt(h)), b1=randn(g, 2 * h, scale=0.1),
             w2=randn(g, h, 2 * h, scale=0.5 / math.sqrt(h)), b2=randn(g, h, scale=0.1))
    p = {k: t.to(dt) for k, t in p.items()}
    p.update(n1w=randn(g, h, scale=0.1, shift=1.0), n1b=randn(g, h, scale=0.1), n2w=randn(g, h, scale=0.1, shift=1.0),
             n2b=randn(g, h, scale=0.1))
    return p


def layer_fp64(x, p):
    F = torch.nn.functional
    h = x.shape[-1]
    u = F.linear(F.layer_norm(x, (h,), p["n1w"], p["n1b"]), p["wi"], p["bi"])
    f, v = u[..., : 2 * h], u[..., 2 * h:]
    a = torch.sigmoid(f)
    fw, bw = [], []
    s = torch.zeros_like(x[:, 0])
    for t in range(x.shape[1]):
        s = a[:, t, :h] * s + (1 - a[:, t, :h]) * v[:, t, :h]
        fw.append(s)
    s = torch.zeros_like(x[:, 0])
    for t in reversed(range(x.shape[1])):
        s = a[:, t, h:] * s + (1 - a[:, t, h:]) * v[:, t, h:]
        bw.append(s)
    y = torch.cat([torch.stack(fw, 1), torch.stack(bw[::-1], 1)], 2)
    x = F.linear(y, p["wo"], p["bo"]) + x
    u = F.gelu(F.linear(F.layer_norm(x, (h,), p["n2w"], p["n2b"]), p["w1"], p["b1"]))
    return F.linear(u, p["w2"], p["b2"]) + x


@pytest.mark.parametrize("dt,tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2)])
def test_layer_of_all_three(dt, tol):
    """a whole encoder layer, forward and every gradient, against fp64 autograd. Relative norms: six roundings to the type in a
    chain of contractions of order one, each at most 2^-8 (2^-24) and random in sign: 6 * 2^-8 = 2.3e-2 (fp32: sums of
    up to 320 terms, (320 / 4 + 16) U = 6e-6 each in a chain of six, partly cancelling)"""
    g = gen(31)
    B, T, h = 5, 37, 160
    x, p, dy = randn(g, B, T, h, dtype=dt), layer_params(g, h, dt), randn(g, B, T, h, dtype=dt)
    names = sorted(p)
    lx = x.clone().requires_grad_(True)
    lp = {k: p[k].clone().requires_grad_(True) for k in names}
    y = layer(lx, lp)
    grads = torch.autograd.grad(y, [lx] + [lp[k] for k in names], dy)
    x64 = x.double().requires_grad_(True)
    p64 = {k: p[k].double().requires_grad_(True) for k in names}
    y64 = layer_fp64(x64, p64)
    g64 = torch.autograd.grad(y64, [x64] + [p64[k] for k in names], dy.double())
    for name, got, ref in zip(["y", "x"] + names, [y.detach()] + list(grads), [y64.detach()] + list(g64)):
        err = float((got.double() - ref).norm() / ref.norm())
        assert err < tol, (name, err)


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
def test_gradients_against_differences(op):
    """central differences of a fp32 scalar loss along random directions: truncation h^2 / 6 of a third derivative of order 1,
    rounding of the loss (sums in fp64 of fp32 outputs of order 1: U sqrt(n) per output) over 2 h"""
    g = gen(41)
    if op == "layer_norm":
        args = [randn(g, 6, 40), randn(g, 40, shift=1.0), randn(g, 40)]
        fn = lambda x, w, b: crnn_hip.layer_norm(x, w, b)  # noqa: E731
    elif op == "linear":
        args = [randn(g, 6, 40), randn(g, 24, 40, scale=0.2), randn(g, 24), randn(g, 6, 24)]
        fn = lambda x, w, b, r: crnn_hip.linear(x, w, b, activation="gelu", residual=r)  # noqa: E731
    else:
        args = [randn(g, 2, 19, 10), randn(g, 2, 19, 10), randn(g, 2, 10)]
        fn = lambda f, v, h: torch.cat([q.flatten() for q in crnn_hip.gated_scan(f, v, h0=h, direction="both", return_state=True)])  # noqa: E731
    leaves = [a.clone().requires_grad_(True) for a in args]
    out = fn(*leaves)
    c = randn(g, *out.shape)
    grads = torch.autograd.grad(out, leaves, c)
    h = 2.0 ** -7
    for i in range(len(args)):
        d = randn(g, *args[i].shape)
        d = d / d.norm()
        with torch.no_grad():
            hi = (fn(*[a + h * d if j == i else a for j, a in enumerate(args)]).double() * c).sum()
            lo = (fn(*[a - h * d if j == i else a for j, a in enumerate(args)]).double() * c).sum()
        num, ana = float((hi - lo) / (2 * h)), float((grads[i].double() * d).sum())
        scale = float(c.norm())
        # third derivative of the outputs along a unit direction: below 20; rounding: 8 U per output of order 4
        assert abs(num - ana) < scale * (20 * h * h / 6 + 32 * U / (2 * h)), (op, i, num, ana)


def test_double_backward_is_refused():
    g = gen(42)
    x = randn(g, 3, 8).requires_grad_(True)
    (gx,) = torch.autograd.grad(crnn_hip.layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.parametrize("dt", TYPES)
def test_results_repeat_bit_for_bit(dt):
    """fixed summation orders: the same call gives the same bits, also beside other work and on another stream"""
    g = gen(51)
    x, p, dy = randn(g, 8, 200, 128, dtype=dt), layer_params(g, 128, dt), randn(g, 8, 200, 128, dtype=dt)
    names = sorted(p)

    def once():
        lx = x.detach().clone().requires_grad_(True)
        lp = {k: p[k].detach().clone().requires_grad_(True) for k in names}
        y = layer(lx, lp)
        return [y.detach()] + list(torch.autograd.grad(y, [lx] + [lp[k] for k in names], dy))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    third = once()   # both streams at once
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_capture_and_replay():
    """a whole layer, forward and backward, captured once and replayed on new inputs between eager runs of its own; two graphs
    of different sizes alive at once (each has its own workspaces)"""
    g = gen(61)
    h = 64
    p = layer_params(g, h, torch.bfloat16)
    names = sorted(p)

    def build(B, T):
        x = randn(g, B, T, h, dtype=torch.bfloat16).requires_grad_(True)
        dy = randn(g, B, T, h, dtype=torch.bfloat16)
        lp = {k: p[k].clone().requires_grad_(True) for k in names}

        def step():
            y = layer(x, lp)
            return [y.detach()] + list(torch.autograd.grad(y, [x] + [lp[k] for k in names], dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, x, dy, step, out
    runs = [build(3, 70), build(1, 2100)]
    for i in range(3):
        for graph, x, dy, step, out in runs:
            with torch.no_grad():
                x.copy_(randn(g, *x.shape))
                dy.copy_(randn(g, *dy.shape))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip([o.clone() for o in out], step()):
                assert torch.equal(a, b), i


def seq_calls(g):
    """name -> (function of a leaf, the leaf) of each operator"""
    w, h = randn(g, 24, 16), randn(g, 2, 16)
    return {"layer_norm": (lambda x: crnn_hip.layer_norm(x), randn(g, 2, 5, 16)),
            "linear": (lambda x: crnn_hip.linear(x, w, activation="gelu"), randn(g, 2, 5, 16)),
            "gated_scan": (lambda x: crnn_hip.gated_scan(x, x, h0=h), randn(g, 2, 5, 16))}


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
def test_forward_mode_is_refused(op):
    """a tangent would be dropped without a word"""
    import torch.autograd.forward_ad as fwAD
    fn, x = seq_calls(gen(62))[op]
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            fn(fwAD.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            fn(fwAD.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
@pytest.mark.parametrize("dt", TYPES)
def test_every_subset_of_gradients(op, dt):
    """whichever inputs want a gradient, each gets what it gets when all do; under no_grad and inference_mode the same output"""
    import itertools
    g = gen(65)
    if op == "layer_norm":
        args, fn = [randn(g, 40, 72, dtype=dt), randn(g, 72), randn(g, 72)], crnn_hip.layer_norm
    elif op == "linear":
        args = [randn(g, 40, 72, dtype=dt), randn(g, 48, 72, dtype=dt), randn(g, 48), randn(g, 40, 48, dtype=dt)]
        fn = lambda x, w, b, r: crnn_hip.linear(x, w, b, activation="silu", residual=r)  # noqa: E731
    else:
        args = [randn(g, 3, 20, 72, dtype=dt), randn(g, 3, 20, 72, dtype=dt), randn(g, 3, 72)]
        fn = lambda f, v, h: crnn_hip.gated_scan(f, v, h0=h)  # noqa: E731
    every = [a.clone().requires_grad_(True) for a in args]
    y = fn(*every)
    dy = randn(g, *y.shape, dtype=dt)
    want = torch.autograd.grad(y, every, dy)
    for k in range(1, len(args)):
        for pick in itertools.combinations(range(len(args)), k):
            leaves = [a.clone().requires_grad_(i in pick) for i, a in enumerate(args)]
            out = fn(*leaves)
            got = torch.autograd.grad(out, [leaves[i] for i in pick], dy)
            assert torch.equal(out, y)
            for i, a in zip(pick, got):
                assert torch.equal(a, want[i]), (pick, i)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert torch.equal(fn(*every), y)


def test_two_threads_at_once():
    """calls from two host threads, each on a stream of its own"""
    import threading
    g = gen(66)
    w, b = randn(g, 96, 64, dtype=torch.bfloat16), randn(g, 96)
    xs = [randn(g, 2, 150, 64, dtype=torch.bfloat16) for _ in range(2)]

    def work(x):
        lx = x.clone().requires_grad_(True)
        y = crnn_hip.linear(crnn_hip.layer_norm(lx), w, b, activation="gelu")
        y = crnn_hip.gated_scan(y, y, direction="both")
        return y.detach(), torch.autograd.grad(y.float().square().sum(), lx)[0]
    want, got = [work(x) for x in xs], [[], []]
    torch.cuda.synchronize()

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i].append(work(xs[i]))
        s.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 5
        for r in got[i]:
            assert torch.equal(r[0], want[i][0]) and torch.equal(r[1], want[i][1])


def test_step_in_place_is_noticed_by_autograd():
    """a graph that saved the state before it was stepped in place must not run on with the new one"""
    g = gen(63)
    f, w, state = randn(g, 3, 8), randn(g, 3, 8).requires_grad_(True), randn(g, 3, 8)
    loss = (state * w).sum()
    crnn_hip.gated_scan_step(f, f, state, out_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
def test_captured_backward_beside_an_eager_graph_of_the_leaf(op):
    """an eager graph of the same leaf, built on the default stream and still alive: the captured backward is refused before
    autograd orders the default stream behind the capture; without that graph the same capture is made"""
    g = gen(64)
    fn, x = seq_calls(g)[op]
    x.requires_grad_(True)
    dy = randn(g, *fn(x).shape)
    (want,) = torch.autograd.grad(fn(x), x, dy)
    held = fn(x)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(fn(x), x, dy)
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(fn(x), x, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        got.zero_()


def test_rows_past_32_bits():
    """row, step and batch offsets past 2^31 elements"""
    big = torch.empty(5 * (1 << 30) // 2, dtype=torch.bfloat16, device=DEV)   # 5 GiB
    ld = (1 << 30) + 16                                                        # the third row starts past 2^31 elements
    g = gen(71)
    x = big.as_strided((3, 72), (ld, 1))
    x.copy_(randn(g, 3, 72))
    small = x.clone()
    assert torch.equal(crnn_hip.layer_norm(x), crnn_hip.layer_norm(small))
    w = randn(g, 40, 72, dtype=torch.bfloat16, scale=0.1)
    xl = big.as_strided((5, 72), ((1 << 29) - 8, 1))   # 1 GiB rows: one row per launch
    xl.copy_(randn(g, 5, 72))
    lw, lx = w.clone().requires_grad_(True), xl.detach().requires_grad_(True)
    dy = randn(g, 5, 40, dtype=torch.bfloat16)
    y = crnn_hip.linear(lx, lw, activation="relu")
    gx, gw = torch.autograd.grad(y, (lx, lw), dy)
    (ry, ey), (rx, ex), (rw, ew), _ = linear_ref(xl, w, None, None, dy, "relu", torch.bfloat16)
    within("y", y, ry, ey)
    within("dx", gx, rx, ex)
    within("dw", gw, rw, ew)
    for f in (big.as_strided((1, 3, 72), (0, ld, 1)), big.as_strided((3, 1, 72), (ld, 0, 1))):
        f.copy_(randn(g, *f.shape))
        c = f.clone()
        assert torch.equal(crnn_hip.gated_scan(f, f), crnn_hip.gated_scan(c, c))
    del big
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ saved-tensor hooks
def strided_calls(g, dt):
    """operator -> (function, leaves), every operand a view whose rows lie apart; the values depend on g alone"""
    wide = lambda *s: randn(g, *s[:-1], 3 * s[-1] + 5, dtype=dt)[..., 1:1 + s[-1]]  # noqa: E731
    return {"layer_norm": (crnn_hip.layer_norm, [wide(6, 7, 70), randn(g, 70), randn(g, 70)]),
            "linear": (lambda x, w, b, r: crnn_hip.linear(x, w, b, activation="gelu", residual=r),
                       [wide(6, 7, 72), wide(48, 72), randn(g, 48), wide(6, 7, 48)]),
            "gated_scan": (lambda f, v, h: crnn_hip.gated_scan(f, v, h0=h, lengths=torch.tensor([9, 4, 0], dtype=torch.int32, device=DEV)),
                           [wide(3, 9, 66), wide(3, 9, 66), randn(g, 3, 66)])}


def spread_out(t):
    """the same values, every element two apart"""
    return torch.stack([t, t], -1)[..., 0]


def turned(t):
    """the same values, the last axis outermost in memory"""
    return t.movedim(-1, 0).contiguous().movedim(0, -1) if t.dim() else t.clone()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
@pytest.mark.parametrize("how", ["host", "compact", "spread", "turned"])
def test_saved_tensor_hooks_may_change_layouts(op, how, dt):
    """what the backward reads comes back from the host compact, or in other strides: the same gradients, bit for bit"""
    fn, args = strided_calls(gen(81), dt)[op]
    leaves = [a.detach().requires_grad_(True) for a in args]
    assert any(not a.is_contiguous() for a in leaves)
    y = fn(*leaves)
    dy = randn(gen(82), *y.shape, dtype=dt)
    want = torch.autograd.grad(y, leaves, dy)
    seen = []
    hooks = {"host": lambda: torch.autograd.graph.save_on_cpu(),
             "compact": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
             "spread": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: seen.append(1) or spread_out(t)),
             "turned": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: seen.append(1) or turned(t))}[how]
    with hooks():
        y2 = fn(*leaves)
    assert torch.equal(y2, y)
    for a, b in zip(torch.autograd.grad(y2, leaves, dy), want):
        assert torch.equal(a, b)
    assert seen or how in ("host", "compact")


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
@pytest.mark.parametrize("what", ["host", "type", "shape"])
def test_saved_tensors_that_do_not_fit_are_refused(op, what):
    """a hook that gives back a tensor of another device, type or shape: an error before anything is launched"""
    fn, args = strided_calls(gen(83), torch.float32)[op]
    leaves = [a.detach().requires_grad_(True) for a in args]
    change = {"host": lambda t: t.cpu(), "type": lambda t: t.double(), "shape": lambda t: t[..., :-1]}[what]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        y = fn(*leaves)
    with pytest.raises(RuntimeError, match=f"{op}: a saved-tensor hook gave back"):
        torch.autograd.grad(y, leaves, torch.ones_like(y))


# ------------------------------------------------------------------------------------------------ the plans of large calls
def linear_plan(m, k, n):
    """(columns of the forward's deep tiles, of the input gradient's, tile of the weight gradient, its splits) of a bf16 product of
    whole vectors, as far as the workspaces tell: a deep kernel copies an operand that is not 16-byte aligned, the others read it
    as it lies, and the weight gradient has a slab a split. 256 or 128 columns by the weighted rounds of the tiles"""
    lib, cu = L.lib(), torch.cuda.get_device_properties(0).multi_processor_count
    k8, n8, at, odd = (k + 7) // 8 * 8, (n + 7) // 8 * 8, 256, 258   # addresses: nothing is read

    def deep(cols, copies):
        rounds = lambda t: -(-(-(-m // 256) * -(-cols // t)) // cu)  # noqa: E731
        return (256 if 7 * rounds(256) <= 5 * rounds(128) else 128) if copies else 0
    fwd = lib.crnn_linear_fwd_workspace(1, odd, k8, at, k8, m, n, k8)
    bwd = lambda x, w, dx, dw: lib.crnn_linear_bwd_workspace(1, at, n8, x, k8, w, k8, 0, dx, dw, 0, m, n8, k8)  # noqa: E731
    slabs = bwd(at, at, 0, 1)
    splits = slabs // (n8 * k8 * 4)
    return (deep(n, fwd), deep(k8, bwd(at, odd, 1, 0)), 256 if bwd(odd, at, 0, 1) > slabs else splits, splits)


# rows, K, N and the plan on 256 CUs: tiles of the forward and of the input gradient (0: register-staged), of the weight gradient
# (256, else its splits: 16 and 15 are those of 128 x 128 tiles, 64 x 64 ones would be cut into 4)
DEEP = [((8192, 512, 1024), (128, 0, 16)),       # whole vectors
        ((8190, 1024, 512), (0, 128, None)),
        ((8195, 509, 1021), (256, 0, 15)),       # copies of x and w for the forward, nothing copied for dx and dw
        ((25601, 261, 250), (128, 256, None)),   # copies throughout; 250 = 31 vectors and two columns
        ((25605, 264, 264), (256, 256, None)),   # row and column remainders of whole vectors
        ((32773, 1531, 765), (256, 256, 256)),   # copies of x, w and dy, remainders everywhere
        ((32768, 768, 1536), (256, 256, 256))]


@pytest.mark.parametrize("size,plan", DEEP)
@pytest.mark.parametrize("kind,bias,res", [("none", None, False), ("gelu", "f32", False), ("silu", "same", True), ("relu", "f32", True),
                                           ("none", "same", True)])
def test_linear_of_large_batches(size, plan, kind, bias, res):
    """the deep kernels with their own epilogue, the copies that they ask for, and the large tiles of the weight gradient; the plan
    is asserted, so that another choice of tiles does not leave them without a test"""
    m, k, n = size
    got = linear_plan(m, k, n)
    assert got[:2] == plan[:2] and plan[2] in (None, got[2]), got
    dt = torch.bfloat16
    g = gen(m + k + n)
    x, w, dy = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=1 / math.sqrt(k)), randn(g, m, n, dtype=dt)
    b = randn(g, n, dtype=torch.float32 if bias == "f32" else dt) if bias else None
    r = randn(g, m, n + 3, dtype=dt)[:, 2:2 + n] if res else None   # rows of odd pitch, 4 bytes off
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = crnn_hip.linear(leaves[0], leaves[1], leaves[2], activation=kind, residual=leaves[3])
    grads = list(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    (ry, ey), (rx, ex), (rw, ew), (rb, eb) = linear_ref(x, w, b, r, dy, kind, dt)
    within("y", y, ry, ey)
    within("dx", grads[0], rx, ex)
    within("dw", grads[1], rw, ew)
    if b is not None:
        within("db", grads[2], rb, eb + ET[b.dtype] * rb.abs())
    if r is not None:
        assert torch.equal(grads[-1], dy)
    with torch.no_grad():
        assert torch.equal(crnn_hip.linear(x, w, b, activation=kind, residual=r), y)
    again = torch.autograd.grad(crnn_hip.linear(leaves[0], leaves[1], leaves[2], activation=kind, residual=leaves[3]),
                                [t for t in leaves if t is not None], dy)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))   # no sum whose order changes


def test_linear_keeps_what_lies_beside_its_rows():
    """the deep kernels' outputs in wider buffers: y, z and dx fill their own columns and rows only"""
    g = gen(91)
    m, k, n, s = 25601, 264, 250, L.stream_ptr()
    assert linear_plan(m, k, n)[:2] == (128, 256)
    x, w, b, res, dy = (randn(g, *q, dtype=torch.bfloat16) for q in ((m, k), (n, k), (n,), (m, n), (m, n)))
    y, z, dx = (torch.full((m + 3, c), 7.0, device=DEV, dtype=torch.bfloat16) for c in (n + 9, n + 6, k + 5))
    need = L.lib().crnn_linear_fwd_workspace(1, x.data_ptr(), k, w.data_ptr(), k, m, n, k)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    L.call("crnn_linear_fwd", 1, x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), 0, 2, res.data_ptr(), n, y.data_ptr(), n + 9, z.data_ptr(),
           n + 6, ws.data_ptr(), need, m, n, k, s)
    need = L.lib().crnn_linear_bwd_workspace(1, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, 2, 1, 0, 0, m, n, k)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    L.call("crnn_linear_bwd", 1, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, z.data_ptr(), n + 6, 2, dx.data_ptr(), k + 5, None, 0, None,
           0, 0, ws.data_ptr(), need, m, n, k, s)
    (ry, ey), (rx, ex), _, _ = linear_ref(x, w, b, res, dy, "gelu", torch.bfloat16)
    rz = x.double() @ w.double().t().contiguous() + b.double()
    ez = (k / 4 + 16) * U * (x.double().abs() @ w.double().abs().t().contiguous() + b.double().abs()) + ET[torch.bfloat16] * rz.abs()
    for name, buf, c, ref, err in (("y", y, n, ry, ey), ("z", z, n, rz, ez), ("dx", dx, k, rx, ex)):
        within(name, buf[:m, :c], ref, err)
        assert (buf[m:] == 7.0).all() and (buf[:m, c:] == 7.0).all(), name


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("off", [0, 1])
def test_linear_in_launches_of_few_rows(dt, off):
    """rows so far apart that a launch's 2 GiB hold 16 of them: 40 rows in launches of 16, 16 and 8, for x (forward and weight gradient),
    then for dy (input and weight gradient), with the pointers of the residual, y and z moved along. off: a pitch that is not a
    whole vector"""
    es = 2 if dt == torch.bfloat16 else 4
    ld = (1 << 27) // es - 8 + off
    big = torch.empty(40 * ld, dtype=dt, device=DEV)
    g = gen(92 + off)
    m, k, n = 40, 72, 56
    x, w, b = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=0.2), randn(g, n)
    res, dy = randn(g, m, n, dtype=dt), randn(g, m, n, dtype=dt)
    far = big.as_strided((m, k), (ld, 1))
    far.copy_(x)
    leaves = [t.detach().requires_grad_(True) for t in (far, w, b, res)]
    y = crnn_hip.linear(leaves[0], leaves[1], leaves[2], activation="silu", residual=leaves[3])
    got = torch.autograd.grad(y, leaves, dy)
    refs = linear_ref(x, w, b, res, dy, "silu", dt)
    for name, a, (ref, err) in zip(("y", "dx", "dw", "db"), (y, got[0], got[1], got[2]), refs):
        within(name, a, ref, err + (U if name == "db" else 0) * ref.abs())
    fdy = big.as_strided((m, n), (ld, 1))
    fdy.copy_(dy)
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(crnn_hip.linear(lx, lw), (lx, lw), fdy)
    refs = linear_ref(x, w, None, None, dy, "none", dt)
    within("dx, far dy", got[0], *refs[1])
    within("dw, far dy", got[1], *refs[2])
    del big, far, fdy, leaves, y
    torch.cuda.empty_cache()


def test_linear_of_more_than_2_gib():
    """x of more than 2 GiB: a launch of the deep kernel over the first 261888 rows and one of the rest"""
    g = gen(93)
    m, k, n = 262144 + 37, 4096, 128
    x = torch.empty(m, k, device=DEV, dtype=torch.bfloat16)
    for i in range(0, m, 65536):
        x[i:i + 65536] = randn(g, min(65536, m - i), k, dtype=torch.bfloat16)
    w, dy = randn(g, n, k, dtype=torch.bfloat16, scale=1 / 64), randn(g, m, n, dtype=torch.bfloat16)
    assert linear_plan(m, k, n)[0] == 128
    leaves = [t.detach().requires_grad_(True) for t in (x, w)]
    y = crnn_hip.linear(*leaves, activation="gelu")
    gx, gw = torch.autograd.grad(y, leaves, dy)
    for lo, hi in ((0, 300), (261888 - 150, 261888 + 150), (m - 300, m)):   # where the launches begin, meet and end
        (ry, ey), (rx, ex), _, _ = linear_ref(x[lo:hi], w, None, None, dy[lo:hi], "gelu", torch.bfloat16)
        within(f"y {lo}", y[lo:hi], ry, ey)
        within(f"dx {lo}", gx[lo:hi], rx, ex)
    # the weight gradient over all rows, in parts: the references add, and so do the bounds (a split of the kernel's sum holds fewer rows
    # than a part, and the parts' bounds on the rounding of their own results add up to no less than the whole's)
    rw, ew = 0, 0
    for i in range(0, m, 65536):
        _, _, (r, e), _ = linear_ref(x[i:i + 65536], w, None, None, dy[i:i + 65536], "gelu", torch.bfloat16)
        rw, ew = rw + r, ew + e
    within("dw", gw, rw, ew)
    del x, dy, y, gx, leaves
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n", [(65600, 40), (32800, 128), (16400, 250), (8200, 512), (8200, 1021), (2100, 2048), (2100, 4001), (2100, 8192),
                                 (2100, 16384), (520, 16390)])
def test_layer_norm_of_more_rows_than_a_grid(m, n, dt):
    """each of the tiles with more rows than its forward's workgroups hold at once (2048 workgroups; wide rows: 512)"""
    g = gen(m + n)
    x, w, b, dy = randn(g, m, n, dtype=dt, shift=0.5), randn(g, n, shift=1.0, scale=0.3), randn(g, n), randn(g, m, n, dtype=dt)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = crnn_hip.layer_norm(*leaves)
    got = [y] + list(torch.autograd.grad(y, leaves, dy))
    for name, a, ref in zip(("y", "dx", "dw", "db"), got, ln_ref(x, w, b, dy, 1e-5, dt)):
        within(name, a, *ref)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("direction", ["forward", "reverse", "both"])
def test_gated_scan_of_many_sequences(direction, dt):
    """1024 rows of channels or more: tiles of four waves, several of them, no segments"""
    g = gen(95)
    b, t, d = 1030, 53, 130
    code = {"forward": 0, "reverse": 1, "both": 2}[direction]
    lib = L.lib()
    assert lib.crnn_gated_scan_workspace(L.dtype_code(dt), b, t, d, code) == 0
    assert lib.crnn_gated_scan_ckpt_bytes(L.dtype_code(dt), b, t, d, code) == b * 4 * d * 4   # four tiles of 16 steps
    f, v, h0 = randn(g, b, t, d, dtype=dt, scale=2.0, shift=1.0), randn(g, b, t, d, dtype=dt), randn(g, b, d)
    scan_check(f, v, h0, None, direction, g, dt)
    lens = torch.randint(0, t + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    lens[:3] = torch.tensor([0, 1, t], device=DEV)
    scan_check(f, v, None, lens, direction, g, dt)


def test_gated_scan_held_steps():
    """infinite logits hold the state: bf16 and fp32 gates are exactly 1 and 0 there, so the state moves only where it enters another
    piece through the composed steps of the piece before. A wave holds 4 steps: of 10 .. 19 the pieces from 12 and from 16 are entered
    that way. The first crossing composes steps 8 .. 11, two of which are not held: A a product of 2 gates that are not 1 (U), H a
    sum of 2 products (4 U max|v|), one multiply-add (2 U), against the same steps walked one by one (the same again); the second composes
    ones and zeros, exactly. Together 14 U max(|h|, |v|), and half a step of the type on each side"""
    for dt in TYPES:
        g = gen(96)
        f, v, h0 = randn(g, 3, 45, 64, dtype=dt), randn(g, 3, 45, 64, dtype=dt), randn(g, 3, 64)
        f[:, 10:20] = float("inf")
        y = crnn_hip.gated_scan(f, v, h0=h0)
        top = float(torch.maximum(v.abs().max().float(), h0.abs().max()))
        held = y[:, 9:10].double().expand(3, 10, 64)
        within("held", y[:, 10:20], held, 14 * U * top + 2 * ET[dt] * held.abs())
        assert torch.equal(y[:, 12:13].expand(3, 8, 64), y[:, 12:20])   # one piece's state, and then the same through ones and zeros


@pytest.mark.parametrize("dt", TYPES)
def test_layer_norm_of_very_wide_rows(dt):
    """a weight gradient over more than 2^27 columns (whose sums in one lane a column of 16 rows would be a grid of 2^32 threads), and the
    statistics of such rows: a lane adds 64 terms at a time and then 2048 of those sums, the workgroup its 1024 lanes, so a sum of n terms is off by
    less than (64 + n / 65536 + 16) U of their magnitudes"""
    g = gen(98)
    m, n = 2, (1 << 27) + 69
    K = (64 + n / 65536 + 64) * U
    x, dy = (torch.empty(m, n, device=DEV, dtype=dt) for _ in range(2))
    for t in (x, dy):
        for i in range(m):
            t[i] = randn(g, n, dtype=dt, shift=0.5)
    w, b = randn(g, n, shift=1.0, scale=0.3), randn(g, n)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = crnn_hip.layer_norm(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, dy)
    y = y.detach()
    # the reference piece by piece of the columns, its sums first
    cols = [slice(i, min(n, i + (1 << 25))) for i in range(0, n, 1 << 25)]
    d = lambda t, c: t[..., c].detach().double()  # noqa: E731
    mean = sum(d(x, c).sum(1, keepdim=True) for c in cols) / n
    rs = 1 / (sum(((d(x, c) - mean) ** 2).sum(1, keepdim=True) for c in cols) / n + 1e-5).sqrt()
    s1, s2, a1, a2 = (sum(f(d(dy, c) * d(w, c), (d(x, c) - mean) * rs).sum(1, keepdim=True) for c in cols) / n
                      for f in (lambda p, q: p, lambda p, q: p * q, lambda p, q: p.abs(), lambda p, q: (p * q).abs()))
    for c in cols:
        xh, dyc, wc = (d(x, c) - mean) * rs, d(dy, c), d(w, c)
        R = 1 + rs * d(x, c).abs().max()
        exh = K * (xh.abs() + R)
        ref = xh * wc + d(b, c)
        within("y", y[:, c], ref, ET[dt] * ref.abs() + exh * wc.abs() + K * (ref.abs() + d(b, c).abs()))
        gg = dyc * wc
        ref = rs * (gg - s1 - xh * s2)
        within("dx", gx[:, c], ref, ET[dt] * ref.abs() + rs * K * (gg.abs() + a1 + xh.abs() * a2 + R * (s2.abs() + xh.abs() * a1)))
        within("dw", gw[c], (dyc * xh).sum(0), (dyc.abs() * exh).sum(0) + 8 * U * (dyc * xh).abs().sum(0))
        within("db", gb[c], dyc.sum(0), 8 * U * dyc.abs().sum(0))
    del x, dy, y, gx, gw, gb, leaves
    torch.cuda.empty_cache()


def test_beside_a_compiled_region_and_under_vmap():
    """torch.compiler.disable keeps an operator out of a compiled function; vmap calls it for each sample"""
    g = gen(99)
    x, w = randn(g, 5, 7, 16), randn(g, 24, 16)
    op = torch.compiler.disable(lambda x: crnn_hip.linear(crnn_hip.layer_norm(x), w))
    want = torch.relu(crnn_hip.linear(crnn_hip.layer_norm(2 * x), w))
    assert torch.equal(torch.compile(lambda x: torch.relu(op(2 * x)), backend="eager")(x), want)
    assert torch.equal(torch.vmap(lambda t: crnn_hip.layer_norm(t))(x), crnn_hip.layer_norm(x))
    assert torch.equal(torch.vmap(lambda t: crnn_hip.gated_scan(t[None], t[None])[0])(x), crnn_hip.gated_scan(x, x))


def test_negated_views():
    """tensors whose memory holds the values' negatives (z.conj().imag): the values count, in inputs and upstream gradients"""
    g = gen(100)
    neg = lambda *s: torch._neg_view(randn(g, *s))  # noqa: E731   (in any layout; z.conj().imag has rows of pairs)
    thin = torch.complex(randn(g, 6, 1), randn(g, 6, 1)).conj().imag
    assert thin.is_neg()
    x, w, f, h, st = neg(6, 16), neg(8, 16), neg(2, 5, 16), neg(2, 16), neg(6, 16)
    for fn, args in ((crnn_hip.layer_norm, (x, w[0], w[1])), (lambda x, w, b, r: crnn_hip.linear(x, w, b, residual=r), (x, w, w[:, 0], neg(6, 8))),
                     (crnn_hip.linear, (thin, neg(8, 1))), (lambda f, h: crnn_hip.gated_scan(f, f, h0=h), (f, h)),
                     (lambda x, s: torch.cat(crnn_hip.gated_scan_step(x, x, s)), (x, st))):
        assert any(a.is_neg() for a in args)
        want = fn(*[a.clone() for a in args])
        assert not any(a.clone().is_neg() for a in args)
        assert torch.equal(fn(*args), want)
    for fn, args in ((crnn_hip.layer_norm, (x,)), (crnn_hip.linear, (x, w)), (crnn_hip.gated_scan, (f, f))):
        leaves = [a.clone().requires_grad_(True) for a in args]
        y = fn(*leaves)
        dy = neg(*y.shape)
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        for a, b in zip(got, torch.autograd.grad(y, leaves, dy.clone())):
            assert torch.equal(a, b)


def test_gated_scan_c_entry_state_gradient_in_place():
    """dh0 over dhT where the sequence has no segments"""
    g = gen(101)
    b, t, d, s = 5, 40, 66, L.stream_ptr()
    lib = L.lib()
    assert lib.crnn_gated_scan_workspace(0, b, t, d, 0) == 0
    f, v, dy, dhT = randn(g, b, t, d), randn(g, b, t, d), randn(g, b, t, d), randn(g, b, d)
    y, ckpt = torch.empty_like(f), torch.empty(lib.crnn_gated_scan_ckpt_bytes(0, b, t, d, 0) // 4, device=DEV)
    L.call("crnn_gated_scan_fwd", 0, f.data_ptr(), t * d, d, v.data_ptr(), t * d, d, None, None, y.data_ptr(), t * d, d, None, ckpt.data_ptr(), None,
           0, b, t, d, 0, s)

    def bwd(din, dout):
        df, dv = torch.empty_like(f), torch.empty_like(f)
        L.call("crnn_gated_scan_bwd", 0, dy.data_ptr(), t * d, d, f.data_ptr(), t * d, d, v.data_ptr(), t * d, d, None, din.data_ptr(),
               ckpt.data_ptr(), df.data_ptr(), t * d, d, dv.data_ptr(), t * d, d, dout.data_ptr(), None, 0, b, t, d, 0, s)
        return df, dv, dout
    same = dhT.clone()
    for a, c in zip(bwd(dhT, torch.empty_like(dhT)), bwd(same, same)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
def test_batched_upstream_gradients_are_refused(op):
    fn, x = seq_calls(gen(102))[op]
    x.requires_grad_(True)
    y = fn(x)
    with pytest.raises(RuntimeError, match=f"{op} runs eagerly"):
        torch.autograd.grad(y, x, torch.ones(3, *y.shape, device=DEV), is_grads_batched=True)


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_layer(reentrant):
    """a layer under activation checkpointing (its saved tensors recomputed in the backward): the same gradients"""
    from torch.utils.checkpoint import checkpoint
    g = gen(103)
    x, p = randn(g, 3, 40, 64, dtype=torch.bfloat16), layer_params(g, 64, torch.bfloat16)
    names = sorted(p)
    dy = randn(g, 3, 40, 64, dtype=torch.bfloat16)

    def grads(run):
        leaves = [x.clone().requires_grad_(True)] + [p[k].clone().requires_grad_(True) for k in names]
        run(lambda x, *w: layer(x, dict(zip(names, w))), leaves).backward(dy)
        return [t.grad for t in leaves]
    for a, b in zip(grads(lambda f, t: checkpoint(f, *t, use_reentrant=reentrant)), grads(lambda f, t: f(*t))):
        assert torch.equal(a, b)


def test_graphed_callables():
    """torch.cuda.make_graphed_callables: forward and backward captured, called in the eager loop with new inputs"""
    g = gen(104)
    p = layer_params(g, 64, torch.bfloat16)
    names = sorted(p)

    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.p = torch.nn.ParameterDict({k: torch.nn.Parameter(p[k].clone()) for k in names})

        def forward(self, x):
            return layer(x, self.p)
    plain, captured = Layer(), Layer()
    sample = randn(g, 3, 40, 64, dtype=torch.bfloat16).requires_grad_(True)
    graphed = torch.cuda.make_graphed_callables(captured, (sample,))
    for _ in range(3):
        x, dy = randn(g, 3, 40, 64, dtype=torch.bfloat16), randn(g, 3, 40, 64, dtype=torch.bfloat16)
        for m, f in ((plain, plain), (captured, graphed)):
            m.zero_grad()
            lx = x.clone().requires_grad_(True)
            f(lx).backward(dy)
            m.gx = lx.grad
        torch.cuda.synchronize()
        assert torch.equal(plain.gx, captured.gx)
        for k in names:
            assert torch.equal(plain.p[k].grad, captured.p[k].grad), k


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan"])
def test_saved_tensors_that_are_wrapped_are_refused(op):
    """a hook that gives back a subclass of its own (no memory of the values behind it), or a sparse tensor"""
    class Wrapped(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.size(), strides=t.stride(), dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            assert func is torch.ops.aten.detach.default   # torch's own, on what a hook returns
            return cls(args[0])
    for change in (Wrapped, lambda t: t.to_sparse()):
        fn, x = seq_calls(gen(105))[op]
        x.requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = fn(x)
        with pytest.raises(RuntimeError, match=f"{op}: a saved-tensor hook gave back a wrapped"):
            torch.autograd.grad(y, x, torch.ones_like(y))
