"""GPU tests of the orthogonalised updates (csrc/ortho.hip): ops.orthogonalize and optim.ClippedMuon against the plain
iteration in 64 bits.

Tolerance.  The iteration amplifies what is rounded in it, float32 or not, so the control is the same iteration in plain
float32 on the host: a kernel product drops one part product of 2^-22 and rounds three times per term where float32's
products round to 2^-24 once, at most a factor 4 per operation, and an operand is held to 2^-22 instead of 2^-24: 8 times
the control's error (relative L2) in all, plus 2^-20 for matrices so small that the control's sums happen to be exact.
The result is rounded to its type once: eps / 2."""
import numpy as np
import pytest
import torch

from tests import _mx4_ref as ref

pytestmark = pytest.mark.gpu


def _matrix(rows, cols, seed, size=1e-3):
    g = torch.Generator().manual_seed(seed)
    k = max(1, min(rows, cols, 8))
    return (torch.randn(rows, cols, generator=g) + 2 * torch.randn(rows, k, generator=g) @
            torch.randn(k, cols, generator=g) / k ** 0.5) * size


def _rel(a, b):
    n = b.double().norm().item()
    return (a.double() - b.double()).norm().item() / n if n else (a.double() - b.double()).norm().item()


def _check(got, g, dtype, steps=5):
    want = ref.orthogonal(g, steps)
    control = _rel(ref.orthogonal(g, steps, dtype=torch.float32), want)
    tol = 8 * control + 2.0 ** -20 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0)
    assert got.dtype == dtype and got.shape == g.shape
    err = _rel(got.cpu(), want)
    assert err <= tol, (tuple(g.shape), err, control)


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (31, 33), (64, 576), (65, 64), (127, 129), (128, 128), (129, 128), (200, 130),
          (256, 1024), (300, 17), (1000, 257), (576, 64), (12, 512), (257, 2304)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_one_matrix_matches_the_iteration(rows, cols, dtype):
    from sln_amodal_amd import ops
    g = _matrix(rows, cols, rows * 10 + cols).to(dtype)
    _check(ops.orthogonalize(g.cuda()), g, dtype)


def test_wide_and_tall_matrices_of_the_classifier():
    from sln_amodal_amd import ops
    g = _matrix(1024, 12544, 1)
    a = ops.orthogonalize(g.cuda())
    _check(a, g, torch.float32)
    # the transpose goes through the same products: the transposed bits
    assert torch.equal(ops.orthogonalize(g.t().contiguous().cuda()), a.t())
    s = torch.linalg.svdvals(a[:, :2048].double().cpu() @ a[:, :2048].double().cpu().t())
    assert torch.isfinite(s).all()


def test_many_matrices_in_one_call_equal_them_alone():
    from sln_amodal_amd import ops
    gs = [_matrix(r, c, i) for i, (r, c) in enumerate(SHAPES * 3)] + [torch.zeros(0, 5), torch.zeros(5, 0)]
    outs = ops.orthogonalize([g.cuda() for g in gs])
    assert isinstance(outs, list)
    for g, o in zip(gs, outs):
        if g.numel():
            _check(o, g, torch.float32)
        else:
            assert o.shape == g.shape
    again = ops.orthogonalize(tuple(g.cuda() for g in gs))
    assert isinstance(again, tuple) and all(torch.equal(a, b) for a, b in zip(outs, again))
    stack = torch.stack([_matrix(48, 80, i) for i in range(6)]).view(2, 3, 48, 80)
    o = ops.orthogonalize(stack.cuda())
    assert o.shape == stack.shape
    for i in range(6):
        _check(o.view(6, 48, 80)[i], stack.view(6, 48, 80)[i], torch.float32)


def test_a_hundred_matrices_take_the_large_tiles():
    from sln_amodal_amd import ops
    gs = [_matrix(*((200, 300) if i % 2 else (300, 200)), seed=i) for i in range(100)]
    outs = ops.orthogonalize([g.cuda() for g in gs])
    for g, o in zip(gs, outs):
        _check(o, g, torch.float32)


@pytest.mark.parametrize("rows,cols", [(64, 576), (33, 577), (32, 1152), (20, 1000), (5, 1153), (63, 65), (32, 32), (1, 3000)])
def test_matrices_that_fit_one_workgroup_and_just_do_not(rows, cols):
    from sln_amodal_amd import ops
    gs = [_matrix(rows, cols, 1), _matrix(cols, rows, 2), _matrix(rows, cols, 3) * 1e-12]
    for o, g in zip(ops.orthogonalize([g.cuda() for g in gs]), gs):
        _check(o, g, torch.float32)


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_steps(steps):
    from sln_amodal_amd import ops
    for rows, cols in ((40, 200), (200, 40)):
        g = _matrix(rows, cols, 3)
        _check(ops.orthogonalize(g.cuda(), steps=steps), g, torch.float32, steps)


def test_sizes_zeros_and_non_finite_values():
    from sln_amodal_amd import ops
    base = _matrix(70, 90, 4, 1.0)
    for size in (1e-30, 1e-6, 1e6, 1e30):                       # eps = 1e-7 counts for the small ones
        g = base * size
        _check(ops.orthogonalize(g.cuda()), g, torch.float32)
    assert not ops.orthogonalize(torch.zeros(70, 90, device="cuda")).any()
    for bad in (float("nan"), float("inf")):
        g = base.clone()
        g[69, 89] = bad
        a, b = ops.orthogonalize([g.cuda(), base.cuda()])
        assert torch.isnan(a).all() and torch.isfinite(b).all()
    # rank one, and one singular value repeated
    u = torch.randn(50, 1) @ torch.randn(1, 60)
    _check(ops.orthogonalize(u.cuda()), u, torch.float32)
    _check(ops.orthogonalize(torch.eye(130).cuda()), torch.eye(130), torch.float32)


def test_strided_matrices():
    from sln_amodal_amd import ops
    base = _matrix(100, 120, 6).cuda()
    for v in (base[3:, 5:], base[::2], base.t(), base[:, ::3], base[:1].expand(4, 120), base[:, :1], base.view(4, 25, 120)[:, 1:]):
        assert torch.equal(ops.orthogonalize(v), ops.orthogonalize(v.contiguous()))


def test_refusals():
    from sln_amodal_amd import ops
    m = torch.zeros(4, 4, device="cuda")
    for err, x, kw in ((TypeError, m.double(), {}), (ValueError, m[0], {}), (ValueError, [m, m.half()], {}),
                       (ValueError, [m[None]], {}), (ValueError, m, {"steps": 0}), (ValueError, m, {"eps": 0.0}),
                       (RuntimeError, m.clone().requires_grad_(), {}), (RuntimeError, [m, m.cpu()], {})):
        with pytest.raises(err):
            ops.orthogonalize(x, **kw)
    with torch.no_grad():
        ops.orthogonalize(m.clone().requires_grad_())


# ------------------------------------------------------------------------------------------------ the optimiser
MATS = [(64, 3, 7, 7), (256, 64, 1, 1), (96, 32, 3, 3), (2, 100), (300, 40), (7, 5, 3), (33, 1), (1, 50), (256, 128, 2, 2)]
VECS = [(64,), (1,), (1023,), (65537,)]


def _plain_step(ps, gs, bs, nm, lr, lr_rest, mu, wd, wd_rest, max_norm, nesterov, dtype):
    norm = sum(float(g.double().pow(2).sum()) for g in gs if g is not None) ** 0.5
    cf = min(1.0, max_norm / (norm + 1e-6))
    out_p, out_b = [], []
    for i, (p, g, b) in enumerate(zip(ps, gs, bs)):
        p, b = p.to(dtype), b.to(dtype)
        if g is not None:
            g = g.to(dtype) * cf
            if i < nm:
                b = mu * b + g
                u = g + mu * b if nesterov else b
                rows, cols = p.shape[0], p.numel() // p.shape[0]
                o = ref.orthogonal(u.reshape(rows, cols), dtype=dtype).reshape(p.shape)
                p = p * (1 - lr * wd) - lr * max(1.0, rows / cols) ** 0.5 * o
            else:
                b = mu * b + (g + wd_rest * p)
                p = p - lr_rest * b
        out_p.append(p)
        out_b.append(b)
    return out_p, out_b, norm


@pytest.mark.parametrize("nesterov,scale", [(True, 1e-4), (True, 1.0), (False, 0.05)])
def test_step_matches_the_formula(nesterov, scale):
    from sln_amodal_amd.optim import ClippedMuon
    g = torch.Generator().manual_seed(1)
    shapes = MATS + VECS
    ps = [torch.randn(s, generator=g) * 0.05 for s in shapes]
    dev = [torch.nn.Parameter(p.cuda()) for p in ps]
    dev[2] = torch.nn.Parameter(ps[2].cuda().contiguous(memory_format=torch.channels_last))
    nm = len(MATS)
    opt = ClippedMuon([{"params": dev[:nm], "weight_decay": 0.1, "orthogonal": True},
                       {"params": dev[nm:], "weight_decay": 1e-3, "lr": 0.05}], lr=0.02, momentum=0.9, nesterov=nesterov)
    bs = [torch.zeros_like(p) for p in ps]
    versions = [p._version for p in dev]
    for r in range(3):
        gs = [torch.randn(s, generator=g) * scale * (1 + i) for i, s in enumerate(shapes)]
        if r == 1:
            gs[3] = gs[nm] = None
        for p, gr in zip(dev, gs):
            p.grad = None if gr is None else gr.cuda()
        args = (ps, gs, bs, nm, 0.02, 0.05, 0.9, 0.1, 1e-3, 5.0, nesterov)
        want_p, want_b, norm = _plain_step(*args, torch.float64)
        ctl_p, _, _ = _plain_step(*args, torch.float32)
        got = opt.step(5.0)
        assert abs(float(got) - norm) <= 2e-7 * norm
        for i, p in enumerate(dev):
            new, old, want = p.detach().cpu().double(), ps[i].double(), want_p[i]
            # the step's own error against the control's, as above, and the rounding of the weights themselves
            step = (want - old).norm().item()
            ctl = (ctl_p[i].double() - want).norm().item()
            assert (new - want).norm().item() <= 8 * ctl + 2.0 ** -20 * step + 2.0 ** -23 * old.norm().item(), (r, i)
            if gs[i] is not None:
                b = opt.state[p].cpu().double()
                assert (b - want_b[i]).norm().item() <= 2.0 ** -21 * (want_b[i].norm().item() + bs[i].norm().item()), (r, i)
        ps = [p.detach().cpu().clone() for p in dev]
        bs = [opt.state[p].cpu().clone() if p in opt.state else torch.zeros_like(q) for p, q in zip(dev, ps)]
    assert all(p._version > v for p, v in zip(dev, versions))


def test_vectors_move_as_under_the_other_optimiser():
    """Without orthogonal groups the step is ClippedSGD's, bit for bit."""
    from sln_amodal_amd.optim import ClippedMuon, ClippedSGD
    g = torch.Generator().manual_seed(2)
    ps = [torch.randn(s, generator=g) for s in VECS + MATS]
    a, b = [[torch.nn.Parameter(p.cuda()) for p in ps] for _ in range(2)]
    oa = ClippedMuon([{"params": a[:3], "weight_decay": 1e-3}, {"params": a[3:]}], lr=0.1, momentum=0.9)
    ob = ClippedSGD([{"params": b[:3], "weight_decay": 1e-3}, {"params": b[3:]}], lr=0.1, momentum=0.9)
    for _ in range(2):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=g).cuda()
            q.grad = p.grad.clone()
        assert float(oa.step(5.0)) == float(ob.step(5.0))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_skipped_steps_write_nothing_and_are_counted():
    from sln_amodal_amd.optim import ClippedMuon
    for with_vectors in (True, False):
        mats = [torch.nn.Parameter(_matrix(40, 60, 1).cuda()), torch.nn.Parameter(_matrix(60, 40, 2).cuda())]
        vecs = [torch.nn.Parameter(torch.ones(9, device="cuda"))] if with_vectors else []
        opt = ClippedMuon([{"params": mats, "orthogonal": True}, {"params": vecs}], lr=0.1, momentum=0.9)
        every = mats + vecs
        for p in every:
            p.grad = torch.randn_like(p)
        opt.step(5.0)
        before = [p.detach().clone() for p in every]
        bufs = [opt.state[p].clone() for p in every]
        same = lambda: all(torch.equal(p, q) for p, q in zip(every, before)) and \
            all(torch.equal(opt.state[p], q) for p, q in zip(every, bufs))
        mats[0].grad[1, 1] = float("inf")
        assert not np.isfinite(float(opt.step(5.0))) and same()
        mats[0].grad[1, 1] = 0.0
        assert np.isfinite(float(opt.step(5.0, veto=torch.ones(1, device="cuda")))) and same()
        assert opt.skipped_steps() == 2 and opt.skipped_clamped_steps() == 1
        opt.step(5.0, veto=torch.zeros(1, device="cuda"))
        assert opt.skipped_steps() == 2 and not same()


def test_state_round_trips_and_hyper_parameters_are_read_at_step_time():
    from sln_amodal_amd.optim import ClippedMuon

    def run(reload_at=None, lr2=None):
        gen = torch.Generator().manual_seed(5)
        dev = [torch.nn.Parameter(torch.randn(s, generator=gen).cuda()) for s in [(20, 30), (30, 20), (30,)]]
        make = lambda lr: ClippedMuon([{"params": dev[:2], "orthogonal": True, "lr": lr}, {"params": dev[2:]}], lr=0.3,
                                      momentum=0.8)
        opt = make(0.1)
        for r in range(3):
            if r == reload_at:
                sd = opt.state_dict()
                opt = make(9.0)
                opt.load_state_dict(sd)
            if r == 1 and lr2:
                opt.param_groups[0]["lr"] = lr2
            for p in dev:
                p.grad = torch.randn(p.shape, generator=gen).cuda()
            opt.step(5.0)
        return [p.detach().clone() for p in dev]

    a = run()
    assert all(torch.equal(p, q) for p, q in zip(a, run(reload_at=2)))
    b = run(lr2=0.01)
    assert not torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


def test_side_streams_and_captured_graphs():
    """Two captured calls share nothing: replayed in turn, with eager calls between, each equals the eager result."""
    from sln_amodal_amd import ops
    xs = [_matrix(96, 300, 1).cuda(), [_matrix(64, 64, 2).cuda(), _matrix(300, 96, 3).cuda()]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for x in xs:
            ops.orthogonalize(x)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.orthogonalize(x))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    flat = lambda o: o if isinstance(o, list) else [o]
    for r in range(3):
        for i, x in enumerate(xs):
            for t in flat(x):
                t.copy_(_matrix(t.shape[0], t.shape[1], 10 * r + i).cuda())
        eager = [flat(ops.orthogonalize(x)) for x in xs]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(flat(o), e))


def test_a_captured_step_replays_beside_eager_ones():
    """The captured step reads its own pointer table: eager steps with other gradients in between do not reach it."""
    from sln_amodal_amd.optim import ClippedMuon

    def make():
        gen = torch.Generator().manual_seed(8)
        ps = [torch.nn.Parameter(torch.randn(s, generator=gen).cuda()) for s in [(20, 30), (100, 130), (30,)]]
        return ps, ClippedMuon([{"params": ps[:2], "orthogonal": True}, {"params": ps[2:]}], lr=0.1, momentum=0.8)

    gen = torch.Generator().manual_seed(9)
    draw = lambda: [torch.randn(s, generator=gen).cuda() for s in [(20, 30), (100, 130), (30,)]]
    a, oa = make()
    b, ob = make()
    static = draw()
    first = draw()
    for ps, opt in ((a, oa), (b, ob)):
        for p, g in zip(ps, first):
            p.grad = g.clone()
        opt.step(5.0)
    torch.cuda.synchronize()
    for p, g in zip(a, static):
        p.grad = g
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            oa.step(5.0)
    torch.cuda.current_stream().wait_stream(s)
    with pytest.raises(RuntimeError):                           # one eager step before each capture
        oa.capturing = True
        oa.step(5.0)
    oa.capturing = False
    for r in range(6):
        new = draw()
        if r % 2 == 0:                                          # a replay against an eager step of the twin
            for g, v in zip(static, new):
                g.copy_(v)
            graph.replay()
        else:                                                   # an eager step of both, the captured gradients left alone
            for p, v in zip(a, new):
                p.grad = v.clone()
            oa.step(5.0)
        for p, v in zip(b, new):
            p.grad = v.clone()
        ob.step(5.0)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), r


@pytest.mark.parametrize("kind", ["ClippedSGD", "ClippedMuon"])
def test_momentum_follows_a_weight_into_another_memory_format(kind):
    """Element i of the momentum is element i of the weight, also after the weight changed to channels-last."""
    from sln_amodal_amd import optim

    def run(change):
        gen = torch.Generator().manual_seed(3)
        p = torch.nn.Parameter(torch.randn(6, 5, 3, 3, generator=gen).cuda())
        groups = [{"params": [p]}]
        if kind == "ClippedMuon":
            groups[0]["orthogonal"] = True
        opt = getattr(optim, kind)(groups, lr=0.1, momentum=0.5)
        for r in range(3):
            if change and r == 1:
                p.data = p.data.contiguous(memory_format=torch.channels_last)
            g = torch.zeros(6, 5, 3, 3)                # (one element per row: no sum depends on the order)
            for i in range(6):
                g[i, i % 5, i // 5, 0] = 1.0 + i
            p.grad = g.cuda()
            opt.step(1e9)
        return p.detach(), opt.state[p]

    (a, ba), (b, bb) = run(False), run(True)
    assert b.is_contiguous(memory_format=torch.channels_last) and not b.is_contiguous()
    assert torch.equal(ba, bb)
    assert torch.equal(a, b)


def test_a_tuple_of_another_type_comes_back_as_a_tuple():
    import collections
    from sln_amodal_amd import ops
    pair = collections.namedtuple("pair", "a b")(torch.randn(4, 6).cuda(), torch.randn(6, 4).cuda())
    out = ops.orthogonalize(pair)
    assert isinstance(out, tuple) and torch.equal(out[0], ops.orthogonalize(pair.a)) and out[1].shape == (6, 4)


# wide and long enough for steps in pairs (the second of a pair takes A from the first one's products)
WIDE = (140, 2700)


def _spectrum(s, seed):
    g = torch.Generator().manual_seed(seed)
    m, n = WIDE
    u = torch.linalg.qr(torch.randn(m, m, generator=g, dtype=torch.double))[0]
    v = torch.linalg.qr(torch.randn(n, m, generator=g, dtype=torch.double))[0]
    return ((u * s) @ v.t()).float()


@pytest.mark.parametrize("kind", ["flat", "linear", "geometric", "outlier", "rank 1", 0.3, 0.1, 0.03, 0.01, 0.003])
def test_steps_in_pairs_over_spectra(kind):
    """A number: half of the singular values are that small beside the others."""
    from sln_amodal_amd import ops
    m = WIDE[0]
    s = torch.ones(m, dtype=torch.double)
    if kind == "linear":
        s = torch.linspace(1, 1 / m, m, dtype=torch.double)
    elif kind == "geometric":
        s = torch.logspace(0, -6, m, dtype=torch.double)
    elif kind == "outlier":
        s[0] = 20.0
    elif kind == "rank 1":
        s[1:] = 0.0
    elif kind != "flat":
        s[m // 2:] = kind
    g = _spectrum(s, 11)
    _check(ops.orthogonalize(g.cuda()), g, torch.float32)
    _check(ops.orthogonalize(g.t().contiguous().cuda()), g.t(), torch.float32)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
def test_steps_in_pairs_any_number(steps):
    from sln_amodal_amd import ops
    g = _matrix(WIDE[0], WIDE[1], steps)
    _check(ops.orthogonalize(g.cuda(), steps=steps), g, torch.float32, steps=steps)


@pytest.mark.parametrize("size", [1e30, 1e-8, 1e-12, 1e-20, 0.0])
def test_steps_in_pairs_of_large_and_tiny_matrices(size):
    """Where eps outweighs the norm the operands are held times a power of two that shrinks from step to step."""
    from sln_amodal_amd import ops
    g = _matrix(WIDE[0], WIDE[1], 7, size)
    _check(ops.orthogonalize(g.cuda()), g, torch.float32)


def test_steps_in_pairs_keep_non_finite_matrices_apart():
    from sln_amodal_amd import ops
    good, bad = _matrix(WIDE[0], WIDE[1], 1), _matrix(WIDE[0], WIDE[1], 2)
    bad[3, 5] = float("inf")
    a, b = ops.orthogonalize([good.cuda(), bad.cuda()])
    _check(a, good, torch.float32)
    assert torch.isnan(b).all()
