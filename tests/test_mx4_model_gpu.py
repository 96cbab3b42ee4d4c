"""The 4-bit classifier head and the orthogonalised update together, as a training run and an evaluation use them: the
head's layers against the plain form, one train step of the assembled model with both, the update of every matrix from the
step's own gradients, the evaluation's kept weight codes."""
import numpy as np
import pytest
import torch

from tests import _mx4_ref as ref

pytestmark = pytest.mark.gpu
LAYERS = r"classifier\.(conv1|conv2|linear_class|linear_bbox)\.weight"


def _model(**kw):
    from sln_amodal_amd import synthetic
    from sln_amodal_amd.config import Config
    from sln_amodal_amd.model import MaskRCNN

    class C(Config):
        NAME = "mx4"
        IMAGE_MAX_DIM = 128
        IMAGE_MIN_DIM = 128
        ARCHITECTURE = "resnet50"

    for k, v in kw.items():
        setattr(C, k, v)
    torch.manual_seed(0)
    cfg = C()
    m = MaskRCNN(cfg, "/tmp/sln_mx4").apply_amodal_heads().cuda()
    m.set_trainable(".*", exclusive_off=False)
    for p in m.GLM_modual.parameters():
        p.requires_grad = False
    batch = synthetic.make_batch(cfg, 2, 128, 128, seed=1, anchors_f64=m.anchors_f64)
    synthetic.calibrate_batchnorm(m, batch["images"])
    synthetic.calibrate_glm(m, batch["images"])
    return m, batch


def _plain_layer(x, w, scale, bias, relu):
    y = ref.values(x) @ ref.values(w).t()
    mag = ref.values(x).abs() @ ref.values(w).abs().t()
    y, mag = y * scale + bias, mag * scale.abs() + bias.abs()
    return (y.clamp(min=0) if relu else y), mag


def test_head_layers_compute_the_rounded_products():
    from sln_amodal_amd import nn_ops
    m, _ = _model(MX4_LAYERS=LAYERS)
    c = m.classifier
    assert all(l.weight._sln_mx4 for l in (c.conv1, c.conv2, c.linear_class, c.linear_bbox))
    assert not m.mask.conv5.weight._sln_mx4
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 256, 7, 7, generator=g).cuda().contiguous(memory_format=torch.channels_last)
    d = lambda t: t.detach().double().cpu()
    with torch.no_grad():
        y1 = nn_ops.conv_bn_act(x, c.conv1, c.bn1, relu=True)
        y2 = nn_ops.conv_bn_act(y1, c.conv2, c.bn2, relu=True)
        y3 = nn_ops.linear(y2.reshape(50, 1024), c.linear_bbox)
    for y, inp, w, conv, bn, relu in (
            (y1, x.permute(0, 2, 3, 1).reshape(50, -1), c.conv1.weight.permute(0, 2, 3, 1).reshape(1024, -1), c.conv1, c.bn1, True),
            (y2, y1.reshape(50, -1), c.conv2.weight.reshape(1024, 1024), c.conv2, c.bn2, True),
            (y3, y2.reshape(50, -1), c.linear_bbox.weight, c.linear_bbox, None, False)):
        scale, bias = torch.ones(w.shape[0], dtype=torch.float64), d(conv.bias)
        if bn is not None:
            s, sh = nn_ops.bn_affine(bn)
            scale, bias = d(s), d(conv.bias) * d(s) + d(sh)
        want, mag = _plain_layer(inp, w, scale, bias, relu)
        K = inp.shape[1]
        assert ((d(y).reshape(50, -1) - want).abs() <= (K + 8) * 2.0 ** -23 * mag + 2.0 ** -24 * want.abs() + 1e-30).all()


def test_evaluation_keeps_the_codes_until_the_weight_changes():
    from sln_amodal_amd import nn_ops
    m, _ = _model(MX4_LAYERS=LAYERS)
    lin = m.classifier.linear_bbox
    x = torch.randn(30, 1024, device="cuda")
    with torch.no_grad():
        a = nn_ops.linear(x, lin)
        codes = lin.weight._sln_mx4_codes[1]
        assert torch.equal(nn_ops.linear(x, lin), a) and lin.weight._sln_mx4_codes[1] is codes
        lin.weight.mul_(-2.0)
        b = nn_ops.linear(x, lin)
        assert lin.weight._sln_mx4_codes[1] is not codes
        # the products are exactly -2 times the first ones; what is added and taken away again is rounded five times
        assert ((b - lin.bias + 2 * (a - lin.bias)).abs() <= 2.0 ** -21 * (a.abs() + b.abs() + lin.bias.abs())).all()
        # a captured call rounds the weight itself: its replays follow the weight
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            nn_ops.linear(x, lin)
            with torch.cuda.graph(g, stream=s):
                out = nn_ops.linear(x, lin)
        torch.cuda.current_stream().wait_stream(s)
        for f in (0.5, -1.0, 4.0):
            lin.weight.mul_(f)
            want = nn_ops.linear(x, lin)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_train_step_with_a_4bit_head_and_orthogonalised_updates():
    """Two optimiser steps of the whole model: gradients everywhere, each matrix moved by lr sqrt(max(1, r / c)) times the
    orthogonal factor of its own clipped, momentum-mixed gradient, biases by SGD; then an evaluation with the new weights."""
    from sln_amodal_amd.optim import ClippedMuon
    m, batch = _model(MX4_LAYERS=LAYERS, OPTIMIZER="muon")
    cfg = m.config
    lr = cfg.LEARNING_RATE
    opt = m.make_optimizer(lr)
    assert isinstance(opt, ClippedMuon)
    watched = {n: p for n, p in m.named_parameters() if p.requires_grad and n in (
        "classifier.conv1.weight", "classifier.conv2.weight", "classifier.linear_bbox.weight", "mask.conv1.weight",
        "fpn.P2_conv1.weight", "classifier.conv2.bias", "fpn.C4.0.conv2.weight")}
    assert len(watched) == 7
    applied = 0
    for step in range(3):
        before = {n: p.detach().double().cpu() for n, p in watched.items()}
        bufs = {n: opt.state[p].double().cpu() if p in opt.state else None for n, p in watched.items()}
        skipped = opt.skipped_steps()
        loss, parts = m.train_step(batch, opt)
        assert torch.isfinite(loss) and all(torch.isfinite(v) for v in parts.values())
        if opt.skipped_steps() != skipped:
            assert all(torch.equal(before[n], p.detach().double().cpu()) for n, p in watched.items())
            continue                                            # (a clamped operand of the other formats: not applied)
        applied += 1
        cf = min(1.0, cfg.GRADIENT_CLIP_NORM / (float(opt.last_norm) + 1e-6))
        for n, p in watched.items():
            g = p.grad.double().cpu() * cf
            now = p.detach().double().cpu()
            if p.dim() < 2:
                b = cfg.LEARNING_MOMENTUM * (bufs[n] if bufs[n] is not None else 0) + g + cfg.WEIGHT_DECAY * before[n]
                want = before[n] - lr * b
                tol = 2.0 ** -22 * before[n].norm() + 2.0 ** -20 * (want - before[n]).norm()
            else:
                mu, big = cfg.MUON_MOMENTUM, lr * cfg.MUON_LR_RATIO
                b = mu * (bufs[n] if bufs[n] is not None else 0) + g
                rows, cols = p.shape[0], p.numel() // p.shape[0]
                u = (g + mu * b).reshape(rows, cols)
                o, o32 = ref.orthogonal(u), ref.orthogonal(u, dtype=torch.float32)
                k = big * max(1.0, rows / cols) ** 0.5
                want = before[n] * (1 - big * cfg.WEIGHT_DECAY) - k * o.reshape(p.shape)
                # 8 times what the iteration loses in plain float32, the clip coefficient's and the weights' roundings
                tol = k * (8 * (o32.double() - o).norm() + 2.0 ** -18 * o.norm()) + 2.0 ** -22 * before[n].norm()
            assert (now - want).norm() <= tol, (step, n, (now - want).norm().item(), float(tol))
    assert applied >= 1
    with torch.no_grad():
        det, mask = m.predict([batch["images"], np.zeros((2, 8 + cfg.NUM_CLASSES)) + [0, 128, 128, 3, 0, 0, 128, 128, 0, 0]],
                              mode="inference")
    assert torch.isfinite(det).all() and torch.isfinite(mask).all()
    assert m.classifier.conv1.weight._sln_mx4_codes[0][0] == m.classifier.conv1.weight._version
