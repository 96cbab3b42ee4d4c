"""Orthogonalised updates on the host: argument checks of the C entries, of ops.orthogonalize and of optim.ClippedMuon, and
the invariants that the fixed operand scale rests on (nothing here launches a kernel)."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import _mx4_ref as ref


def test_the_iteration_keeps_singular_values_inside_the_fixed_operand_range():
    """p maps [0, 1.21] into itself and its factor a + b l + c l^2 stays below 3.4445 + rounding on l in [0, 1.21^2]: with
    the scale 2^14 no operand reaches fp16's largest value 65504."""
    a, b, c = ref.NS
    s = np.linspace(0, 1.21, 200001)
    p = a * s + b * s ** 3 + c * s ** 5
    assert p.min() >= 0 and p.max() <= 1.21
    q = a + b * s ** 2 + c * s ** 4
    assert np.abs(q).max() <= 3.4446 and 3.4446 * 2 ** 14 < 65504
    # ... and five steps bring (0.005, 1] into [0.67, 1.21]
    s = np.linspace(0.005, 1, 100001)
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert 0.67 <= s.min() and s.max() <= 1.21


def test_entries_check_their_arguments():
    from sln_amodal_amd import _lib
    from sln_amodal_amd.ops import _OrthoDesc
    from sln_amodal_amd.optim import _MuonDesc
    L = _lib.lib()
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 255) // 256 * 256
    vp = C.c_void_p(p)
    small = (_OrthoDesc * 1)((p, p, 8, 8, 4, 8))
    assert L.sln_orthogonalize_workspace_bytes(small, 1) == 0   # runs on one CU, without a workspace
    d = (_OrthoDesc * 2)((p, p, 99, 99, 70, 99), (0, 0, 0, 0, 0, 5))
    need = L.sln_orthogonalize_workspace_bytes(d, 2)
    assert need > 0 and L.sln_orthogonalize_workspace_bytes(d, 0) == 0
    run = lambda descs, n, dtype=0, steps=5, eps=1e-7, ws=vp, nbytes=1 << 30: L.sln_orthogonalize(
        descs, n, dtype, steps, eps, ws, nbytes, None)
    assert run(d, 2, dtype=7) == 1 and run(d, 2, steps=0) == 1 and run(d, 2, steps=65) == 1
    assert run(d, 2, eps=0.0) == 1 and run(d, 2, eps=float("nan")) == 1 and run(None, 2) == 1 and run(d, -1) == 1
    assert run(d, 2, ws=None) == 1 and run(d, 2, ws=C.c_void_p(p + 8)) == 1
    assert run(d, 2, nbytes=need - 1) == 2
    assert run(d, 0) == 0                                       # nothing to do
    assert run((_OrthoDesc * 1)((0, 0, 0, 0, 0, 5)), 1) == 0
    assert run((_OrthoDesc * 1)((0, p, 8, 8, 4, 8)), 1) == 1
    assert run((_OrthoDesc * 1)((p, p, 7, 8, 4, 8)), 1) == 1
    assert run((_OrthoDesc * 1)((p, p, 8, 7, 4, 8)), 1) == 1
    assert run((_OrthoDesc * 1)((p, p, 70000, 70000, 70000, 70000)), 1) == 4
    assert run((_OrthoDesc * 1)((p, p, 8, 8, -4, 8)), 1) == 1
    m = (_MuonDesc * 1)((p, p, p, 70, 80, 0.1, 1.0))
    need = L.sln_muon_step_workspace_bytes(m, 1)
    step = lambda descs, sq=vp, ws=vp, nbytes=1 << 30: L.sln_muon_step_f32(descs, 1, 5, 1e-7, sq, 5.0, 0.9, 1, ws, nbytes,
                                                                           None)
    assert step(m, sq=None) == 1 and step(m, ws=None) == 1 and step(m, nbytes=need - 1) == 2
    assert step((_MuonDesc * 1)((p, 0, p, 70, 80, 0.1, 1.0))) == 1


def test_wrong_calls_are_refused():
    from sln_amodal_amd import ops
    from sln_amodal_amd.optim import ClippedMuon
    with pytest.raises(RuntimeError):
        ops.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        ops.orthogonalize(3)
    m, v = torch.nn.Parameter(torch.zeros(4, 4)), torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError):
        ClippedMuon([{"params": [v], "orthogonal": True}], lr=0.1)
    with pytest.raises(ValueError):
        ClippedMuon([{"params": [m], "orthogonal": True}, {"params": [m]}], lr=0.1)
    with pytest.raises(ValueError):
        ClippedMuon([{"params": [m], "orthogonal": True}], lr=0.1, steps=0)
    opt = ClippedMuon([{"params": [m], "orthogonal": True}, {"params": [v], "lr": 0.5}], lr=0.1, momentum=0.9)
    assert opt.lr == 0.5 and opt.momentum == 0.9 and opt.step(5.0) is None         # no gradients: nothing to do
    m.grad, v.grad = torch.ones(4, 4), torch.ones(4)
    with pytest.raises(RuntimeError):
        opt.step(5.0)
    sd = opt.state_dict()
    sd["param_groups"][0]["orthogonal"] = False
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)


def test_model_makes_the_configured_optimiser():
    from sln_amodal_amd.config import Config
    assert Config.OPTIMIZER in ("sgd", "muon") and Config.MX4_LAYERS == ""


def test_model_tags_and_groups():
    """The configuration's layers are tagged (also the ones that the head surgery replaces), a layer that is no product of
    rows is refused, and OPTIMIZER = "muon" puts every matrix into the orthogonal group."""
    from sln_amodal_amd.config import Config
    from sln_amodal_amd.model import MaskRCNN

    class Cfg(Config):
        NAME = "tags"
        IMAGE_MAX_DIM = 128
        ARCHITECTURE = "resnet50"
        OPTIMIZER = "muon"
        MX4_LAYERS = r"classifier\.(conv2|linear_class)\.weight"

    m = MaskRCNN(Cfg(), "/tmp/sln_tags").apply_amodal_heads(glm=False)
    tagged = sorted(n for n, p in m.named_parameters() if getattr(p, "_sln_mx4", False))
    assert tagged == ["classifier.conv2.weight", "classifier.linear_class.weight"]
    assert m.set_mx4_layers("") == 0 and not m.classifier.conv2.weight._sln_mx4
    assert m.set_mx4_layers(r"classifier\..*") == 4
    for bad in (r"mask\.conv5\.weight", r"fpn\..*", ".*"):
        with pytest.raises(ValueError):
            m.set_mx4_layers(bad)
    assert m.classifier.conv2.weight._sln_mx4                   # a refused pattern changes nothing
    opt = m.make_optimizer(0.001)
    for g in opt.param_groups:
        assert all((p.dim() >= 2) == g["orthogonal"] for p in g["params"])
    n = sum(len(g["params"]) for g in opt.param_groups)
    assert n == sum(p.requires_grad for p in m.parameters())
    assert [g["lr"] for g in opt.param_groups] == [0.02, 0.001, 0.001]
    m.config.OPTIMIZER = "adam"
    with pytest.raises(ValueError):
        m.make_optimizer(0.001)


def test_matrices_longer_than_the_entries_take_are_refused_when_the_optimiser_is_made():
    from sln_amodal_amd.optim import ClippedMuon
    p = torch.nn.Parameter(torch.empty(1, (1 << 22) + 1, device="meta"))
    with pytest.raises(ValueError):
        ClippedMuon([{"params": [p], "orthogonal": True}], lr=0.1)
    ClippedMuon([{"params": [torch.nn.Parameter(torch.empty(1, 1 << 22, device="meta"))], "orthogonal": True}], lr=0.1)
