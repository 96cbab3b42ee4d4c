"""Hyper-parameters of the optimisers' groups (no kernel runs)."""
import pytest
import torch
from torch import nn


def _muon(lr=0.001, ratio=20.0):
    from sln_amodal_amd.optim import ClippedMuon
    m, v, w = nn.Parameter(torch.zeros(4, 4)), nn.Parameter(torch.zeros(4)), nn.Parameter(torch.zeros(3))
    return ClippedMuon([{"params": [m], "orthogonal": True, "lr": ratio * lr}, {"params": [v]}, {"params": [w]}], lr=lr)


def _rates(opt):
    return [g["lr"] for g in opt.param_groups]


def test_setting_the_rate_keeps_the_ratio_of_the_groups():
    opt = _muon()
    opt.lr *= 0.1
    assert opt.lr == pytest.approx(1e-4, rel=1e-15) and _rates(opt) == pytest.approx([2e-3, 1e-4, 1e-4], rel=1e-15)
    opt.lr = 0.5
    assert _rates(opt) == pytest.approx([10.0, 0.5, 0.5], rel=1e-15)
    opt.param_groups[0]["lr"] = 1.0                             # a ratio set by hand is the one that is kept
    opt.lr = 0.25
    assert _rates(opt) == [0.5, 0.25, 0.25]


def test_the_ratio_survives_a_rate_of_zero_and_a_reload():
    opt = _muon()
    opt.lr = 0.0
    assert _rates(opt) == [0.0, 0.0, 0.0]
    other = _muon()
    other.load_state_dict(opt.state_dict())
    for o in (opt, other):
        o.lr = 0.002
        assert _rates(o) == pytest.approx([0.04, 0.002, 0.002], rel=1e-15)
    bad = _muon()
    for g in bad.param_groups:
        g["lr"] = 0.0                                           # set by hand: nothing to scale from
    with pytest.raises(ValueError):
        bad.lr = 0.1
    assert _rates(bad) == [0.0, 0.0, 0.0]


def test_groups_that_disagree_are_brought_together():
    opt = _muon()
    opt.param_groups[2]["lr"] = 0.004
    with pytest.raises(ValueError):
        opt.lr
    opt.lr = 0.002
    assert _rates(opt) == pytest.approx([0.04, 0.002, 0.002], rel=1e-15)


def test_orthogonal_groups_alone():
    from sln_amodal_amd.optim import ClippedMuon
    a, b = nn.Parameter(torch.zeros(4, 4)), nn.Parameter(torch.zeros(4, 5))
    opt = ClippedMuon([{"params": [a], "orthogonal": True}, {"params": [b], "orthogonal": True, "lr": 0.4}], lr=0.1)
    opt.lr = 0.2
    assert _rates(opt) == [0.2, 0.8] and opt.lr == 0.2


def test_one_rate_for_all_groups_of_the_other_optimiser():
    from sln_amodal_amd.optim import ClippedSGD
    a, b = nn.Parameter(torch.zeros(4)), nn.Parameter(torch.zeros(5))
    opt = ClippedSGD([{"params": [a]}, {"params": [b], "lr": 0.4}], lr=0.1)
    opt.lr = 0.2
    assert _rates(opt) == [0.2, 0.2]
