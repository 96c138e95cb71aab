"""RCNN(rnn_type="glr"): the gated-linear-recurrence stack in the BiLSTM's place (crnn_hip/glr.py), on the engine, in training
(run_training, checkpoints, resume) and in inference."""
import csv
import os

import pytest
import torch

from crnn_hip.ctc import ctc_loss
from model.model import RCNN

DEV = "cuda"


def stack_fp64(x, p, nl):
    """the stack as crnn_hip/glr.py writes it, in fp64, step by step"""
    F = torch.nn.functional
    for l in range(nl):
        q = {k.split(f"enc_rnn.{l}.", 1)[1]: v for k, v in p.items() if k.startswith(f"enc_rnn.{l}.")}
        if "proj.weight" in q:
            x = F.linear(x, q["proj.weight"], q["proj.bias"])
        h = x.shape[-1]
        u = F.linear(F.layer_norm(x, (h,), q["norm1.weight"], q["norm1.bias"]), q["in.weight"], q["in.bias"])
        f, v = u[..., : 2 * h], u[..., 2 * h:]
        a = torch.sigmoid(f)
        outs = []
        for lo, order in ((0, range(x.shape[1])), (h, reversed(range(x.shape[1])))):
            s, col = torch.zeros_like(x[:, 0]), {}
            for t in order:
                at = a[:, t, lo:lo + h]
                s = at * s + (1 - at) * v[:, t, lo:lo + h]
                col[t] = s
            outs.append(torch.stack([col[t] for t in range(x.shape[1])], 1))
        x = x + F.linear(torch.cat(outs, 2), q["out.weight"], q["out.bias"])
        g = F.gelu(F.linear(F.layer_norm(x, (h,), q["norm2.weight"], q["norm2.bias"]), q["ff1.weight"], q["ff1.bias"]))
        x = x + F.linear(g, q["ff2.weight"], q["ff2.bias"])
    return x


def make(hidden, dtype, nl=2, decoder="ctc", drop=0.0, seed=5):
    torch.manual_seed(seed)
    return RCNN(num_classes=40, hidden_size=hidden, num_rnn_layers=nl, compute_dtype=dtype, blank_id=None, rnn_type="glr",
                decoder=decoder, enc_dropout_p=drop)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,B,T", [(64, 3, 32), (36, 2, 17), (512, 8, 128)])
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 5e-5), (torch.bfloat16, 7e-2)])
def test_stack_matches_fp64(hidden, B, T, dtype, tol):
    """output, input gradient and every parameter gradient of two layers in relative norm. bf16: 9 stored roundings per layer and
    direction in a chain, each at most 2^-8 of what it rounds: 18 * 2^-8 = 7e-2; the packed weights are the same on both
    sides (the reference takes their bf16 values). fp32: sums of up to 1024 terms, (1024 / 4 + 16) 2^-24 = 1.6e-5 of the sum of
    magnitudes, three times that for what cancels"""
    m = make(hidden, dtype).to(DEV).train()
    m.flatten_parameters_()
    with torch.no_grad():
        for k, v in m.named_parameters():
            if k.startswith("enc_rnn.") and v.dim() == 2:
                v.copy_(v.to(dtype).float())   # representable, so that the packed copies are exact
    eng = m._engine_for(torch.zeros(1, 3, 32, 8, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(B, T, 512, generator=g, device=DEV).to(dtype).float()
    dout = torch.randn(B, T, hidden, generator=g, device=DEV).to(dtype).float()
    grads, _, _ = m._grad_views()
    y, dx = eng.bilstm_stack(x, dout, grads)
    p = {k: v.detach().double().requires_grad_(True) for k, v in m.named_parameters() if k.startswith("enc_rnn.")}
    x64 = x.double().requires_grad_(True)
    y64 = stack_fp64(x64, p, 2)
    y64.backward(dout.double())
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y, y64.detach()) < tol and rel(dx, x64.grad) < tol
    for k, v in p.items():
        assert rel(grads[k], v.grad) < tol, (k, rel(grads[k], v.grad))
    again = eng.bilstm_stack(x)   # inference: nothing kept for a backward, the same numbers
    assert torch.equal(again, y)


@pytest.mark.gpu
def test_lines_of_many_lengths_share_the_scratch():
    """batches of other geometries: the same results as a fresh engine's, and one scratch buffer, not one a size"""
    def engine():
        m = make(64, torch.bfloat16).to(DEV).train()
        m.flatten_parameters_()
        return m, m._engine_for(torch.zeros(1, 3, 32, 8, device=DEV))
    m, eng = engine()
    g = torch.Generator(device=DEV).manual_seed(10)
    grads, _, _ = m._grad_views()
    for B, T in ((2, 40), (1, 700), (5, 9), (2, 40)):
        x, dout = torch.randn(B, T, 512, generator=g, device=DEV), torch.randn(B, T, 64, generator=g, device=DEV)
        y, dx = eng.bilstm_stack(x, dout, grads)
        m2, fresh = engine()
        grads2, _, _ = m2._grad_views()
        y2, dx2 = fresh.bilstm_stack(x, dout, grads2)
        assert torch.equal(y, y2) and torch.equal(dx, dx2)
        for k in grads:
            if k.startswith("enc_rnn."):
                assert torch.equal(grads[k], grads2[k]), k
    assert len([k for k in eng.ws.bufs if k.startswith("glr.ws")]) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_model_trains_end_to_end(dtype):
    """the whole model: every parameter gets its gradient, a second backward accumulates, eval agrees with train"""
    m = make(64, dtype).to(DEV).train()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 3, 32, 128, generator=g).to(DEV)
    tg = torch.randint(1, 40, (4, 5), generator=g).to(DEV)
    tl = torch.tensor([5, 3, 1, 4]).to(DEV)
    ctc_loss(m(x), tg, tl).backward()
    first = {k: p.grad.clone() for k, p in m.named_parameters()}
    for k, v in first.items():
        assert torch.isfinite(v).all() and v.any(), k
    ctc_loss(m(x), tg, tl).backward()   # running statistics moved, batch statistics did not: the same gradient once more
    for k, p in m.named_parameters():
        if k.startswith("enc_rnn."):
            err = float((p.grad - 2 * first[k]).norm() / (2 * first[k]).norm())
            assert err < 1e-6, (k, err)
    m.eval()
    with torch.no_grad():
        lg = m(x)
        assert lg.shape == (4, 16, 40) and torch.isfinite(lg).all()
        assert torch.equal(m(x), lg)
        assert m.encode(x).shape == (4, 16, 64)


@pytest.mark.gpu
def test_attention_head_on_the_stack():
    m = make(64, torch.bfloat16, decoder="attn").to(DEV).train()
    x = torch.randn(2, 3, 32, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    text = torch.ones(2, 9, dtype=torch.long, device=DEV)
    m(x, text=text, is_train=True, batch_max_length=8).square().mean().backward()
    for k, p in m.named_parameters():
        assert torch.isfinite(p.grad).all(), k
    assert m.cnn.conv0[0].weight.grad.any() and getattr(m.enc_rnn[0], "in").weight.grad.any()
    with torch.no_grad():
        assert m.eval()(x, is_train=False, batch_max_length=8).shape == (2, 9, 40)


@pytest.mark.gpu
def test_run_training_checkpoint_resume_and_inference(tmp_path):
    """config key "rnn_type": trained, saved, resumed, and the checkpoint opened by OCRInference with the stack it holds"""
    from inference import OCRInference
    from test_train_api import CHARSET, LINES, _cfg
    from training.train import run_training
    cfg = _cfg(tmp_path, rnn_type="glr", epochs=1)
    out = run_training(cfg, device="cuda")
    assert 0.0 <= out["val_acc"] <= 1.0 and out["val_loss"] < float("inf")
    last = os.path.join(cfg.exp_dir, "last_ckpt.pth")
    ck = torch.load(last, map_location="cpu", weights_only=True)
    assert ck["config"]["rnn_type"] == "glr" and "enc_rnn.1.ff2.bias" in ck["model_state"]
    run_training(_cfg(tmp_path, rnn_type="glr", epochs=2, resume_path=last), device="cuda")
    rows = list(csv.reader(open(os.path.join(cfg.exp_dir, "metrics_epoch.csv"), encoding="utf-8")))
    assert [r[0] for r in rows[1:]] == ["1", "2"]
    ocr = OCRInference(last, CHARSET, device="cuda", img_h=32, img_w=128)
    assert ocr.model.rnn_type == "glr"
    assert isinstance(ocr.predict(os.path.join(LINES, "a", "img_000.png")), str)


def test_surface_and_state_dict():
    """names, shapes and the choice of the stack; the default model is unchanged"""
    m = make(64, torch.float32)
    sd = m.state_dict()
    assert tuple(sd["enc_rnn.0.proj.weight"].shape) == (64, 512) and "enc_rnn.1.proj.weight" not in sd
    assert tuple(sd["enc_rnn.1.in.weight"].shape) == (256, 64) and tuple(sd["enc_rnn.1.out.weight"].shape) == (64, 128)
    assert "enc_rnn.0.proj.weight" not in make(512, torch.float32).state_dict()
    from training.utils import rcnn_from_state
    again = rcnn_from_state(sd, 40, 64, 1, 2, 0, None)
    assert again.rnn_type == "glr" and again.num_rnn_layers == 2
    for k, v in again.state_dict().items():
        assert torch.equal(v, sd[k])
    assert rcnn_from_state(RCNN(num_classes=40, hidden_size=64).state_dict(), 40, 64, 1, 2, 0, None).rnn_type == "lstm"
    with pytest.raises(ValueError, match="rnn_type"):
        RCNN(num_classes=40, rnn_type="gru")
    with pytest.raises(RuntimeError, match="HIP device"):
        m(torch.zeros(1, 3, 32, 64))
