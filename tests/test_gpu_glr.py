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


# ------------------------------------------------------------------------------------------------ data parallel
def _shard(rank):
    from crnn_hip.recipe import synthetic_batch
    x, _, tg, tl = synthetic_batch(8, 32, 128, 8, 40, seed=200 + rank)
    return x.to(DEV), tg, tl


def _flat_model(seed):
    m = make(64, torch.bfloat16, seed=seed).to(DEV).train()
    m.flatten_parameters_()
    return m


def _dp_worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank),
                      CRNN_SHARE_DEVICE="1", HSA_ENABLE_IPC_MODE_LEGACY="0")
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    sys.path.insert(0, os.path.join(here, "../rcnn-ocr_amd"))
    import torch.distributed as dist
    try:
        from crnn_hip import dist as D
        from crnn_hip.engine import CRNNEngine
        from crnn_hip.optim import FusedAdamW
        D.init_from_env("gloo")
        torch.cuda.set_device(0)
        m = _flat_model(5 + rank)              # other weights on rank 1: the broadcast has to replace them
        flat = m._flat_param.detach().cpu()    # (gloo: host tensors only)
        D.broadcast_params(flat)
        with torch.no_grad():
            m._flat_param.copy_(flat)
        m.mark_params_changed()
        opt = FusedAdamW(m, lr=1e-3)
        opt.zero_grad()
        # the reducer as in deployment, on a host copy of the flat gradient that the hook fills with what each stage reports final
        offs, host = m.flat_offsets(), torch.full_like(flat, float("nan"))
        red = D.OverlappedAllReduce(host, offs, min_bucket_bytes=1 << 20)
        stages = []

        def hook(prefixes):
            stages.append(list(prefixes))
            for k, (s, n) in offs.items():
                if k.startswith(tuple(prefixes)):
                    host[s:s + n].copy_(m._flat_grad[s:s + n])
            red.ready(prefixes)
        m.stage_done = hook
        x, tg, tl = _shard(rank)
        ctc_loss(m(x), tg, tl).backward()
        red.finish()
        spans = sorted(red.last_issued)
        tiled = len(spans) > 1 and spans[0][0] == 0 and spans[-1][1] == host.numel() and all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
        m._flat_grad.copy_(host)
        opt.step(grad_scale=1.0 / world)
        torch.cuda.synchronize()
        q.put((rank, None, stages == CRNNEngine.backward_stages(), tiled, host.numpy(), m._flat_param.detach().cpu().numpy()))
    except Exception:   # report to the parent instead of hanging it
        import traceback
        q.put((rank, traceback.format_exc(), False, False, None, None))
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


@pytest.mark.gpu
def test_data_parallel_of_the_stack():
    """two processes on the one GPU, a shard each: the stages report their gradients final in order, the buckets tile the flat
    gradient, the reduced gradient is the sum of the shards' own, bit for bit, and both replicas take the same step as one process with
    that sum"""
    import socket

    import torch.multiprocessing as mp

    from crnn_hip.optim import FusedAdamW
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ps = [ctx.Process(target=_dp_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in ps:
        p.start()
    res = sorted((q.get(timeout=100) for _ in ps), key=lambda r: r[0])
    for p in ps:
        p.join(timeout=30)
    for r in res:
        assert r[1] is None, r[1]
        assert r[2] and r[3]
    m = _flat_model(5)
    opt = FusedAdamW(m, lr=1e-3)
    grads = []
    for rank in range(2):
        opt.zero_grad()
        x, tg, tl = _shard(rank)
        ctc_loss(m(x), tg, tl).backward()
        grads.append(m._flat_grad.detach().clone())
    m._flat_grad.copy_(grads[0] + grads[1])
    for _, p in m.named_parameters():
        assert p.grad is not None
    opt.step(grad_scale=0.5)
    want_g, want_p = (grads[0] + grads[1]).cpu(), m._flat_param.detach().cpu()
    for r in res:
        assert torch.equal(torch.from_numpy(r[4]), want_g)
        assert torch.equal(torch.from_numpy(r[5]), want_p)


@pytest.mark.gpu
def test_stack_at_the_training_batch():
    """256 lines of 32 frames at hidden 512, the batch at which the products run on their large tiles: output, input gradient and
    parameter gradients against fp64, and a second backward that adds to the first's gradients in fp32. The bound of
    test_stack_matches_fp64: 9 stored roundings per layer and direction in a chain, each at most 2^-8 of what it rounds"""
    m = make(512, torch.bfloat16).to(DEV).train()
    m.flatten_parameters_()
    with torch.no_grad():
        for k, v in m.named_parameters():
            if k.startswith("enc_rnn.") and v.dim() == 2:
                v.copy_(v.bfloat16().float())
    eng = m._engine_for(torch.zeros(1, 3, 32, 8, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(12)
    x, dout = (torch.randn(256, 32, 512, generator=g, device=DEV).bfloat16().float() for _ in range(2))
    grads, _, _ = m._grad_views()
    y, dx = eng.bilstm_stack(x, dout, grads)
    p = {k: v.detach().double().requires_grad_(True) for k, v in m.named_parameters() if k.startswith("enc_rnn.")}
    x64 = x.double().requires_grad_(True)
    y64 = stack_fp64(x64, p, 2)
    y64.backward(dout.double())
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y, y64.detach()) < 7e-2 and rel(dx, x64.grad) < 7e-2
    for k, v in p.items():
        assert rel(grads[k], v.grad) < 7e-2, (k, rel(grads[k], v.grad))
    first = {k: grads[k].clone() for k in p}
    xs, ds = x.bfloat16(), dout.bfloat16()
    _, saved = eng._rnn_forward(xs, 256, 32, True)
    eng._rnn_backward(ds, saved, 256, 32, 1)
    for k in p:
        assert torch.equal(grads[k], first[k] + first[k]), k
