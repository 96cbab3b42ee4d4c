"""Optimiser steps over matrices whose Gram products are cut and whose Newton-Schulz steps go in pairs, weights written by the
last product.  Tolerances as in test_ortho_gpu.test_step_matches_the_formula."""
import pytest
import torch

from tests.test_ortho_gpu import _plain_step

pytestmark = pytest.mark.gpu
WIDE = [(140, 300, 3, 3), (2600, 130), (100, 4000), (64, 100), (300, 2700), (257, 2561)]
VECS = [(64,), (1023,)]


def test_these_matrices_are_cut_and_paired():
    """The rules of csrc/ortho.hip (ortho_plan): no square products from 81 k-steps of 32 on, pairs where the sum of m^2 n is
    over twice that of m^3; a contraction of 80 k-steps is cut where there are fewer tiles than CUs."""
    sides = [(min(s[0], n), max(s[0], n)) for s in WIDE for n in [int(torch.Size(s[1:]).numel())]]
    assert max(-(-n // 32) for _, n in sides) > 80
    assert sum(m * m * n for m, n in sides) > 2 * sum(m ** 3 for m, _ in sides)
    assert sum((-(-m // 128)) * (-(-m // 128) + 1) // 2 for m, _ in sides) < 64


@pytest.mark.parametrize("nesterov,scale", [(True, 1e-4), (True, 1.0), (False, 0.05)])
def test_wide_matrices_step_by_the_formula(nesterov, scale):
    from sln_amodal_amd.optim import ClippedMuon
    g = torch.Generator().manual_seed(1)
    shapes, nm = WIDE + VECS, len(WIDE)
    ps = [torch.randn(s, generator=g) * 0.05 for s in shapes]
    dev = [torch.nn.Parameter(p.cuda()) for p in ps]
    opt = ClippedMuon([{"params": dev[:nm], "weight_decay": 0.1, "orthogonal": True},
                       {"params": dev[nm:], "weight_decay": 1e-3, "lr": 0.05}], lr=0.02, momentum=0.9, nesterov=nesterov)
    bs = [torch.zeros_like(p) for p in ps]
    for r in range(2):
        gs = [torch.randn(s, generator=g) * scale * (1 + i) for i, s in enumerate(shapes)]
        for p, gr in zip(dev, gs):
            p.grad = gr.cuda()
        args = (ps, gs, bs, nm, 0.02, 0.05, 0.9, 0.1, 1e-3, 5.0, nesterov)
        want_p, want_b, norm = _plain_step(*args, torch.float64)
        ctl_p, _, _ = _plain_step(*args, torch.float32)
        assert abs(float(opt.step(5.0)) - norm) <= 2e-7 * norm
        for i, p in enumerate(dev):
            new, old, want = p.detach().cpu().double(), ps[i].double(), want_p[i]
            step, ctl = (want - old).norm().item(), (ctl_p[i].double() - want).norm().item()
            assert (new - want).norm().item() <= 8 * ctl + 2.0 ** -20 * step + 2.0 ** -23 * old.norm().item(), (r, i)
            b = opt.state[p].cpu().double()
            assert (b - want_b[i]).norm().item() <= 2.0 ** -21 * (want_b[i].norm().item() + bs[i].double().norm().item()), (r, i)
        ps = [p.detach().cpu().clone() for p in dev]
        bs = [opt.state[p].cpu().clone() for p in dev]
    # a vetoed step writes nothing
    before = [p.detach().clone() for p in dev]
    opt.step(5.0, veto=torch.ones(1, device="cuda"))
    assert all(torch.equal(p, q) for p, q in zip(dev, before)) and opt.skipped_steps() == 1
