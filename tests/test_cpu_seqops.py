"""The sequence operators' refusals (crnn_hip.layer_norm, linear, gated_scan), without a GPU: the Python entry points check
their arguments before they ask for a device, and the C entry points check theirs before they launch anything."""
import ctypes as C

import pytest
import torch

import crnn_hip
from crnn_hip import _lib as L

X = torch.zeros(4, 6)
F3 = torch.zeros(2, 5, 6)


@pytest.mark.parametrize("call", [
    lambda: crnn_hip.layer_norm(X.half()),
    lambda: crnn_hip.layer_norm(X.double()),
    lambda: crnn_hip.layer_norm(torch.zeros(())),
    lambda: crnn_hip.layer_norm(torch.zeros(3, 0)),
    lambda: crnn_hip.layer_norm(X, torch.ones(5)),
    lambda: crnn_hip.layer_norm(X, torch.ones(6).bfloat16()),
    lambda: crnn_hip.layer_norm(X, torch.ones(6), torch.ones(6, 1)),
    lambda: crnn_hip.layer_norm(X, eps=-1.0),
    lambda: crnn_hip.layer_norm(X, eps=float("nan")),
    lambda: crnn_hip.linear(X.half(), torch.zeros(3, 6).half()),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6).bfloat16()),
    lambda: crnn_hip.linear(X, torch.zeros(3, 7)),
    lambda: crnn_hip.linear(X, torch.zeros(6)),
    lambda: crnn_hip.linear(X, torch.zeros(0, 6)),
    lambda: crnn_hip.linear(torch.zeros(4, 0), torch.zeros(3, 0)),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6), torch.zeros(4)),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6), torch.zeros(3).bfloat16()),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6), activation="tanh"),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6), residual=torch.zeros(3)),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6), residual=torch.zeros(4, 3).bfloat16()),
    lambda: crnn_hip.gated_scan(X, X),
    lambda: crnn_hip.gated_scan(F3.half(), F3.half()),
    lambda: crnn_hip.gated_scan(F3, F3.bfloat16()),
    lambda: crnn_hip.gated_scan(F3, F3[:, :4]),
    lambda: crnn_hip.gated_scan(F3, F3, direction="backward"),
    lambda: crnn_hip.gated_scan(F3[..., :5], F3[..., :5], direction="both"),
    lambda: crnn_hip.gated_scan(F3, F3, h0=torch.zeros(2, 5)),
    lambda: crnn_hip.gated_scan(F3, F3, h0=torch.zeros(2, 6).bfloat16()),
    lambda: crnn_hip.gated_scan(F3, F3, lengths=torch.ones(3, dtype=torch.int32)),
    lambda: crnn_hip.gated_scan(F3, F3, lengths=torch.ones(2)),
    lambda: crnn_hip.gated_scan(F3, F3, lengths=[1, 2]),
    lambda: crnn_hip.layer_norm(torch.zeros(1).expand(1 << 31)),
    lambda: crnn_hip.linear(torch.zeros(1).expand(1, 1 << 31), torch.zeros(1).expand(1, 1 << 31)),
    lambda: crnn_hip.gated_scan(torch.zeros(1).expand(1, 1 << 31, 1), torch.zeros(1).expand(1, 1 << 31, 1)),
    lambda: crnn_hip.gated_scan_step(F3, F3, F3),
    lambda: crnn_hip.gated_scan_step(X, X, X[:2]),
    lambda: crnn_hip.gated_scan_step(X, X, X.bfloat16()),
    lambda: crnn_hip.gated_scan_step(X, X, X, out_state=torch.zeros(6, 4).t()),
])
def test_bad_arguments_raise_value_error(call):
    with pytest.raises(ValueError):
        call()


def test_step_refuses_overlapping_states_and_gradients():
    buf = torch.zeros(30)
    a, b = buf[:24].view(4, 6), buf[6:].view(4, 6)
    with pytest.raises(ValueError, match="overlaps"):
        crnn_hip.gated_scan_step(X, X, a, out_state=b)
    with pytest.raises(RuntimeError, match="inference only"):
        crnn_hip.gated_scan_step(X.clone().requires_grad_(True), X, X)


def test_step_refuses_an_output_that_is_an_input_or_a_leaf():
    """out_state over f or v would be written while they are read; a leaf that wants a gradient is not written in place"""
    buf = torch.zeros(60)
    for i, lo in enumerate((0, 12, 23)):
        f = buf[lo:lo + 24].view(4, 6)
        with pytest.raises(ValueError, match="f or v"):
            crnn_hip.gated_scan_step(*((f, X) if i % 2 else (X, f)), X, out_state=buf[:24].view(4, 6))
    with pytest.raises(RuntimeError, match="HIP device"):      # beside it: the call gets as far as asking for a device
        crnn_hip.gated_scan_step(buf[24:48].view(4, 6), X, X, out_state=buf[:24].view(4, 6))
    with pytest.raises(RuntimeError, match="inference only"):
        crnn_hip.gated_scan_step(X, X, X, out_state=torch.zeros(4, 6, requires_grad=True))


@pytest.mark.parametrize("call", [
    lambda: crnn_hip.layer_norm(X),
    lambda: crnn_hip.linear(X, torch.zeros(3, 6)),
    lambda: crnn_hip.gated_scan(F3, F3),
    lambda: crnn_hip.gated_scan_step(X, X, X),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="HIP device"):
        call()


def test_binding_is_required(monkeypatch):
    """the operators are in libcrnn_torch.so, and a missing one raises instead of falling back"""
    ops = L.ops()
    for name in ("layer_norm", "linear", "gated_scan", "gated_scan_step"):
        assert hasattr(ops, name)
    monkeypatch.setattr(L, "_ops", None)
    monkeypatch.setattr(L, "TORCH_LIB_PATH", "/nonexistent/libcrnn_torch.so")
    with pytest.raises(RuntimeError, match="not built"):
        L.ops()


P = C.c_void_p(256)   # never dereferenced: every call below is refused before a launch


def _refused(name, *args, match):
    with pytest.raises(RuntimeError, match=match):
        L.call(name, *args)


def test_c_layernorm_refusals():
    ok = (0, P, 8, None, None, P, 8, None, None, 4, 8, 1e-5, None)

    def bad(match, **kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        _refused("crnn_layernorm_fwd", *a, match=match)
    bad("dtype", _0=2)
    bad("ld >= N", _2=7)
    bad("ld >= N", _6=7)
    bad("N <= 2", _10=0)
    bad("N <= 2", _10=(1 << 30) + 1, _2=1 << 31, _6=1 << 31)
    bad("M >= 0", _9=-1)
    bad("go together", _7=P)
    bad("null", _1=None)
    assert L.lib().crnn_layernorm_fwd(0, None, 8, None, None, None, 8, None, None, 0, 8, 1e-5, None) == 0   # no rows
    need = L.lib().crnn_layernorm_bwd_workspace(0, 4, 8)
    assert need > 0
    _refused("crnn_layernorm_bwd", 0, P, 8, P, 8, None, P, P, None, 0, P, 8, P, P, 0, P, need - 1, 4, 8, None, match="workspace")
    _refused("crnn_layernorm_bwd", 0, P, 8, P, 8, None, None, P, None, 0, P, 8, None, None, 0, None, 0, 4, 8, None, match="null")
    _refused("crnn_layernorm_bwd", 0, P, 8, P, 8, None, P, P, P, 4, P, 8, None, None, 0, None, 0, 4, 8, None, match="ld >= N")


def test_c_linear_refusals():
    lib = L.lib()
    # the deep kernels (256 rows a tile, three quarters of the CUs or more) take whole aligned vectors only: others are copied
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert lib.crnn_linear_fwd_workspace(1, P, 264, P, 264, 25600, 256, 264) == 0
    assert lib.crnn_linear_fwd_workspace(1, P, 257, P, 257, 25600, 256, 257) == up(25600 * 264 * 2) + up(256 * 264 * 2)
    assert lib.crnn_linear_fwd_workspace(1, C.c_void_p(258), 264, P, 264, 25600, 256, 264) == up(25600 * 264 * 2)
    # the register-staged ones, fp32 and the few-row kernel read them as they lie
    assert lib.crnn_linear_fwd_workspace(1, P, 257, P, 257, 1000, 256, 257) == 0
    assert lib.crnn_linear_fwd_workspace(0, P, 257, P, 257, 25600, 256, 257) == 0
    assert lib.crnn_linear_fwd_workspace(1, P, 257, P, 257, 32, 256, 257) == 0

    def fwd(match, dt=1, x=P, ldx=16, ldw=16, act=0, res=None, ldr=0, ldy=8, z=None, ldz=0, ws=None, n=0, M=99, N=8, K=16):
        _refused("crnn_linear_fwd", dt, x, ldx, P, ldw, None, 0, act, res, ldr, P, ldy, z, ldz, ws, n, M, N, K, None, match=match)
    fwd("dtype", dt=2)
    fwd("act", act=4)
    fwd("act", act=-1)
    fwd("N, K >= 1", N=0)
    fwd("M >= 0", M=-1)
    fwd("row stride", ldx=15)
    fwd("row stride", ldw=15)
    fwd("row stride", ldy=7)
    fwd("row stride", z=P, ldz=7)
    fwd("row stride", res=P, ldr=7)
    fwd("null", x=None)
    big = dict(M=25600, N=256, K=264, ldx=265, ldw=264, ldy=256)
    fwd("workspace", ws=P, n=1, **big)
    fwd("workspace", **big)
    fwd("2 GiB", ldw=1 << 28)
    assert lib.crnn_linear_fwd(1, None, 16, None, 16, None, 0, 0, None, 0, None, 8, None, 0, None, 0, 0, 8, 16, None) == 0

    def bwd(match, lddy=8, z=None, ldz=0, act=0, dw=P, dw_f32=1, acc=0, n=1 << 20, M=4, x=P):
        _refused("crnn_linear_bwd", 1, P, lddy, x, 16, P, 16, z, ldz, act, P, 16, dw, dw_f32, P, 1, acc, P, n, M, 8, 16, None,
                 match=match)
    bwd("row stride", lddy=7)
    bwd("row stride", act=2, z=P, ldz=7)
    bwd("null", act=2, ldz=8)
    bwd("null", x=None)
    bwd("accumulate", dw_f32=0, acc=1)
    bwd("workspace", n=0)


def test_c_gated_scan_refusals():
    lib = L.lib()
    assert lib.crnn_gated_scan_workspace(1, 256, 32, 1024, 2) == 0      # enough rows: no segments
    seg = lib.crnn_gated_scan_workspace(1, 1, 16384, 64, 0)             # one long sequence: segment summaries
    assert seg > 0 and lib.crnn_gated_scan_ckpt_bytes(1, 1, 16384, 64, 0) > 0
    assert lib.crnn_gated_scan_workspace(1, 1, 1, 64, 0) == 0

    def fwd(match, dt=1, f=P, h0=None, hT=None, ws=None, n=0, B=1, T=8, D=64, dr=0):
        _refused("crnn_gated_scan_fwd", dt, f, T * D, D, P, T * D, D, h0, None, P, T * D, D, hT, None, ws, n, B, T, D, dr, None,
                 match=match)
    fwd("dtype", dt=2)
    fwd("dir", dr=3)
    fwd("even D", dr=2, D=63)
    fwd("B/T/D", T=-1)
    fwd("null", f=None)
    fwd("workspace", T=16384)
    fwd("workspace", T=16384, ws=P, n=seg - 1)
    fwd("hT == h0", T=16384, ws=P, n=seg, h0=P, hT=P)
    for b, t, d in ((0, 8, 64), (1, 8, 0), (1, 0, 64)):                 # nothing to do
        assert lib.crnn_gated_scan_fwd(1, None, 0, 0, None, 0, 0, None, None, None, 0, 0, None, None, None, 0, b, t, d, 0, None) == 0
    _refused("crnn_gated_scan_bwd", 1, P, 64, 64, P, 64, 64, P, 64, 64, None, None, None, P, 64, 64, P, 64, 64, None, None, 0, 1, 1,
             64, 0, None, match="null")


def _operators(x):
    """the four entry points on one [4, 6] input"""
    return {"layer_norm": lambda: crnn_hip.layer_norm(x), "linear": lambda: crnn_hip.linear(x, torch.zeros(3, 6)),
            "gated_scan": lambda: crnn_hip.gated_scan(x[None], x[None]), "gated_scan_step": lambda: crnn_hip.gated_scan_step(x, x, x)[0]}


@pytest.mark.parametrize("op", ["layer_norm", "linear", "gated_scan", "gated_scan_step"])
def test_tracing_and_transforms_are_refused(op):
    """they run eagerly on plain tensors: a trace would hold the results' allocation and not the kernel that fills them"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    with FakeTensorMode(), pytest.raises(RuntimeError, match=f"{op} runs eagerly"):
        _operators(torch.zeros(4, 6))[op]()
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(RuntimeError, match=f"{op} runs eagerly"):
            make_fx(lambda x: _operators(x)[op](), tracing_mode=mode)(X)
    with pytest.raises(RuntimeError, match=f"{op} runs eagerly"):
        torch.func.grad(lambda x: _operators(x)[op]().sum())(X)
    with pytest.raises(Exception, match=f"{op} runs eagerly"):
        torch.compile(lambda x: _operators(x)[op]() + 1, backend="eager")(X)

    class Count(TorchDispatchMode):   # a mode that only watches does not stand in the way: the call gets as far as the device
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Count(), pytest.raises(RuntimeError, match="HIP device"):
        _operators(X)[op]()


def test_step_refuses_a_negated_output():
    with pytest.raises(ValueError, match="negated"):
        crnn_hip.gated_scan_step(X, X, X, out_state=torch._neg_view(torch.zeros(4, 6)))


def test_c_gated_scan_bwd_refuses_a_state_gradient_over_its_input():
    """segments run at once: the first one's dh0 may not be written over the dhT that the others still read"""
    lib = L.lib()
    seg = lib.crnn_gated_scan_workspace(1, 1, 16384, 64, 0)
    assert seg > 0

    def bwd(match, n=seg, dhT=P, dh0=P):
        _refused("crnn_gated_scan_bwd", 1, P, 64, 64, P, 64, 64, P, 64, 64, None, dhT, P, P, 64, 64, P, 64, 64, dh0, P, n, 1, 16384, 64, 0, None,
                 match=match)
    bwd("dh0 == dhT")
    bwd("workspace", n=seg - 1)


def test_c_layernorm_bwd_refuses_dx_over_dres_of_another_pitch():
    _refused("crnn_layernorm_bwd", 0, P, 8, P, 8, None, P, P, P, 9, P, 8, None, None, 0, None, 0, 4, 8, None, match="same row stride")
