"""GPU tests of optimiser steps that are captured into graphs beside what goes on eagerly: what layers keep of the weights, what
the graphs' launches read, and what the optimiser's state does meanwhile.  Every comparison is for equal bits: a captured
step is the same launches over the same values."""
import copy
import gc
import pickle
import weakref

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
KINDS = ["ClippedSGD", "ClippedMuon"]


def _make(kind, shapes, seed=8):
    from sln_amodal_amd import optim
    gen = torch.Generator().manual_seed(seed)
    ps = [nn.Parameter((torch.randn(s, generator=gen) * 0.1).cuda()) for s in shapes]
    return ps, _optimiser(kind, ps)


def _optimiser(kind, ps, lr=0.1):
    from sln_amodal_amd import optim
    if kind == "ClippedSGD":
        return optim.ClippedSGD([{"params": ps, "weight_decay": 1e-3}], lr=lr, momentum=0.8)
    mats, rest = [p for p in ps if p.dim() > 1], [p for p in ps if p.dim() < 2]
    return optim.ClippedMuon([{"params": mats, "orthogonal": True}, {"params": rest}], lr=lr, momentum=0.8)


def _grads(ps, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(p.shape, generator=gen).cuda() for p in ps]


def _set(ps, gs):
    for p, g in zip(ps, gs):
        p.grad = g


def _capture(opt, **kw):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            opt.step(5.0, **kw)
    torch.cuda.current_stream().wait_stream(s)
    return graph


@pytest.mark.parametrize("kind", KINDS)
def test_a_4_bit_layer_sees_the_weights_that_replays_wrote(kind):
    """Evaluate (the weight's codes are kept), replay a captured step, evaluate again: the codes of the new weight."""
    from sln_amodal_amd import nn_ops, ops
    lin = nn.Linear(96, 40).cuda()
    lin.weight._sln_mx4 = True
    ps = [lin.weight, lin.bias]
    opt = _optimiser(kind, ps)
    x = _grads([torch.empty(30, 96)], 1)[0]
    static = _grads(ps, 2)
    _set(ps, static)
    fresh = lambda: ops.mx4_linear(x, lin.weight.detach().clone(), lin.bias.detach().clone())
    with torch.no_grad():
        first = nn_ops.linear(x, lin)
        opt.step(5.0)
        assert torch.equal(nn_ops.linear(x, lin), fresh())
        graph = _capture(opt)
        assert torch.equal(nn_ops.linear(x, lin), fresh())       # (kept here, were the weight not in a captured step)
        for r in range(3):
            for g, v in zip(static, _grads(ps, 10 + r)):
                g.copy_(v)
            graph.replay()
            y = nn_ops.linear(x, lin)
            assert torch.equal(y, fresh()) and not torch.equal(y, first), r
            first = y


def test_other_layers_see_them_after_replayed():
    from sln_amodal_amd import nn_ops
    conv = nn.Conv2d(64, 64, 3, padding=1).cuda()
    ps = list(conv.parameters())
    opt = _optimiser("ClippedSGD", ps)
    x = _grads([torch.empty(1, 64, 16, 16)], 1)[0].contiguous(memory_format=torch.channels_last)
    static = _grads(ps, 2)
    _set(ps, static)

    def fresh():                                                 # the same layer as a new module: nothing kept
        other = nn.Conv2d(64, 64, 3, padding=1).cuda()
        other.load_state_dict(conv.state_dict())
        return nn_ops.conv_bn_act(x, other)

    with torch.no_grad():
        first = nn_ops.conv_bn_act(x, conv)
        opt.step(5.0)
        graph = _capture(opt)
        nn_ops.conv_bn_act(x, conv)
        for r in range(3):
            for g, v in zip(static, _grads(ps, 10 + r)):
                g.copy_(v)
            graph.replay()
            opt.replayed()
            y, want = nn_ops.conv_bn_act(x, conv), fresh()
            # (operand scales are kept per layer: equal up to their choice, 2^-20 of the largest; stale weights are O(1) off)
            assert (y - want).abs().max() <= 1e-4 * want.abs().max() and (y - first).abs().max() > 1e-2 * want.abs().max(), r
            first = y


def test_replayed_moves_the_versions_of_captured_weights_only():
    ps, opt = _make("ClippedSGD", [(20, 30), (30,)])
    other = nn.Parameter(torch.ones(3, device="cuda"))
    opt.param_groups[0]["params"].append(other)
    versions = [p._version for p in ps + [other]]
    opt.replayed()
    assert versions == [p._version for p in ps + [other]]
    _set(ps, _grads(ps, 3))
    opt.step(5.0)
    _capture(opt)
    versions = [p._version for p in ps + [other]]
    opt.replayed()
    assert [p._version for p in ps + [other]] == [versions[0] + 1, versions[1] + 1, versions[2]]


SHAPES = [(20, 30), (100, 130), (30,)]


def _twins(kind):
    (a, oa), (b, ob) = _make(kind, SHAPES), _make(kind, SHAPES)
    first = _grads(a, 9)
    for ps, opt in ((a, oa), (b, ob)):
        _set(ps, [g.clone() for g in first])
        opt.step(5.0)
    return a, oa, b, ob


def _same(a, oa, b, ob):
    torch.cuda.synchronize()
    return all(torch.equal(p, q) for p, q in zip(a, b)) and \
        all(torch.equal(oa.state[p], ob.state[q]) for p, q in zip(a, b))


def _churn():
    """Takes over what the allocator got back: small blocks full of ones."""
    return [torch.full((n,), -1, dtype=torch.int64, device="cuda") for n in (1, 2, 3, 4, 6, 8, 9, 16, 32, 64) for _ in range(20)]


@pytest.mark.parametrize("kind", KINDS)
def test_what_a_captured_step_reads_outlives_eager_steps_of_another_set(kind):
    """An eager step without one of the gradients, and one with another weight decay, make new plans: the graph keeps its own."""
    a, oa, b, ob = _twins(kind)
    static = _grads(a, 20)
    _set(a, static)
    graph = _capture(oa)
    kept = [weakref.ref(t) for t in oa._plan] + [weakref.ref(t) for t in oa.state.values()]
    for change in ("set", "decay"):
        for ps, opt in ((a, oa), (b, ob)):
            _set(ps, [g.clone() for g in _grads(ps, 30)])
            if change == "set":
                ps[0].grad = None
            else:
                opt.param_groups[-1]["weight_decay"] = 0.25
            opt.step(5.0)
            opt.param_groups[-1]["weight_decay"] = 1e-3 if kind == "ClippedSGD" else 0.0
    gc.collect()
    assert all(r() is not None for r in kept)                     # (from the host, before any replay)
    assert _same(a, oa, b, ob)
    ones = _churn()
    for r in range(3):
        new = _grads(a, 40 + r)
        for g, v in zip(static, new):
            g.copy_(v)
        graph.replay()
        _set(b, [v.clone() for v in new])
        ob.step(5.0)
        assert _same(a, oa, b, ob), r
    assert all((t == -1).all() for t in ones)


@pytest.mark.parametrize("kind", KINDS)
def test_loaded_momentum_reaches_a_captured_step(kind):
    a, oa, b, ob = _twins(kind)
    static = _grads(a, 20)
    _set(a, static)
    graph = _capture(oa)
    addresses = [oa.state[p].data_ptr() for p in a]
    saved = [p.detach().clone() for p in a]
    sd = oa.state_dict()
    sd["state"] = {i: {"momentum_buffer": s["momentum_buffer"].clone()} for i, s in sd["state"].items()}
    for without in (None, 2):                                     # the whole state; one without a buffer: zeros
        if without is not None:
            sd["state"].pop(without)
        graph.replay()
        for ps, opt in ((a, oa), (b, ob)):
            with torch.no_grad():
                for p, v in zip(ps, saved):
                    p.copy_(v)
            opt.load_state_dict(sd)
        if without is not None:
            ob.state[b[without]] = torch.zeros_like(b[without])
        assert [oa.state[p].data_ptr() for p in a] == addresses and _same(a, oa, b, ob)
        new = _grads(a, 50)
        for g, v in zip(static, new):
            g.copy_(v)
        graph.replay()
        _set(b, [v.clone() for v in new])
        ob.step(5.0)
        assert _same(a, oa, b, ob)


@pytest.mark.parametrize("kind", KINDS)
def test_captures_that_would_take_memory_of_the_capture_are_refused(kind):
    ps, opt = _make(kind, [(6, 5, 3, 3), (20, 30), (20, 30)])
    _set(ps, _grads(ps, 3))
    before = [p.detach().clone() for p in ps]

    def refused():
        opt.capturing = True                                      # (what a capture sets; nothing is being captured here)
        with pytest.raises(RuntimeError, match="eager step"):
            opt.step(5.0)
        opt.capturing = False

    refused()                                                     # no eager step yet
    ps[2].grad = None
    opt.step(5.0)
    before = [p.detach().clone() for p in ps]
    _set(ps, _grads(ps, 4))
    ps[1].grad = None
    refused()                                                     # as many weights of the same sizes, but not the same ones
    _set(ps, _grads(ps, 4))
    refused()                                                     # more of them
    assert all(torch.equal(p, q) for p, q in zip(ps, before))
    opt.step(5.0)
    graph = _capture(opt)
    ps[0].data = ps[0].data.contiguous(memory_format=torch.channels_last)
    _set(ps, _grads(ps, 5))
    with pytest.raises(RuntimeError, match="memory format"):      # the graph writes this weight's momentum
        opt.step(5.0)
    del graph



@pytest.mark.parametrize("kind", KINDS)
def test_replays_count_their_vetoes(kind):
    """The first veto of all comes inside of the capture: its counter was there before."""
    a, oa, _, _ = _twins(kind)
    _set(a, _grads(a, 20))
    veto = torch.zeros(1, device="cuda")
    graph = _capture(oa, veto=veto)
    for hit in (1, 0, 1, 1):
        veto.fill_(hit)
        before = [p.detach().clone() for p in a]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, before)) == bool(hit)
    assert oa.skipped_clamped_steps() == 3 and oa.skipped_steps() == 3


@pytest.mark.parametrize("kind", KINDS)
def test_captures_in_a_row(kind):
    """Several steps captured after one eager step, each with gradients of its own, replayed out of order."""
    a, oa, b, ob = _twins(kind)
    statics, graphs = [], []
    for i in range(8):
        statics.append(_grads(a, 20 + i))
        _set(a, statics[-1])
        graphs.append(_capture(oa))
    for r, i in enumerate((3, 0, 7, 3, 5, 1)):
        new = _grads(a, 60 + r)
        for g, v in zip(statics[i], new):
            g.copy_(v)
        graphs[i].replay()
        _set(b, [v.clone() for v in new])
        ob.step(5.0)
        assert _same(a, oa, b, ob), (r, i)
    _set(a, _grads(a, 90))
    oa.capturing = True
    with pytest.raises(RuntimeError, match="nothing is being captured"):
        oa.step(5.0)


@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_step_outlives_its_optimiser(kind):
    """The graph is replayed after the optimiser went: what it reads hangs on the weights."""
    a, oa, b, ob = _twins(kind)
    static = _grads(a, 20)
    _set(a, static)
    graph = _capture(oa)
    kept = [weakref.ref(t) for t in oa._plan] + [weakref.ref(t) for t in oa.state.values()]
    for clone in (pickle.loads(pickle.dumps(a[0])), copy.deepcopy(a[0])):
        assert not getattr(clone, "_sln_captured", None) and torch.equal(clone, a[0])
    momentum = [oa.state[p] for p in a]
    del oa
    gc.collect()
    assert all(r() is not None for r in kept)                     # (from the host, before any replay)
    ones = _churn()
    for r in range(3):
        new = _grads(a, 40 + r)
        for g, v in zip(static, new):
            g.copy_(v)
        graph.replay()
        _set(b, [v.clone() for v in new])
        ob.step(5.0)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and \
            all(torch.equal(m, ob.state[q]) for m, q in zip(momentum, b)), r
    assert all((t == -1).all() for t in ones)
