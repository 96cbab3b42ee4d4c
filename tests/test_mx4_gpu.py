"""GPU tests of the microscaled 4-bit row products (csrc/mx4.hip, csrc/mx4_grad.hip) against the plain 64-bit form.

Tolerances.  Rounding: none, codes and scales have to be equal.  Products: every product of two rounded values is exact, a
float32 sum of n terms is off by at most one unit in the last place (2^-23) of the sum of magnitudes per addition, so
n 2^-23 sum|a b| bounds any order of it; the result is rounded once more (eps / 2).  Where all sums are exactly
representable the bits have to be equal."""
import numpy as np
import pytest
import torch

from tests import _mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _x(shape, seed, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))).to(dtype)


def _check_codes(q, x):
    codes, scales = ref.unpack(q)
    want, ws = ref.round_codes(x.detach().double().cpu().numpy())
    assert np.array_equal(scales, ws)
    # (a negative value that rounds to zero may carry the sign bit or not: the same value)
    zero = (want & 7) == 0
    assert np.array_equal(np.where(zero, 0, codes & 7), np.where(zero, 0, want & 7))
    assert np.array_equal(codes[~zero], want[~zero])
    return ref.code_values(codes, scales, x.shape[-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 255), (4, 256), (7, 257), (33, 1003), (130, 12544)])
def test_rounding_equals_the_definition(R, K, dtype):
    from sln_amodal_amd import ops
    x = _x((R, K), R * 1000 + K, dtype)
    q = ops.mx4_quantize(x.cuda())
    v = _check_codes(q, x)
    for t in TYPES:
        assert torch.equal(q.dequantize(t).cpu(), torch.from_numpy(v).to(t))
    assert q.dequantize().dtype == dtype and tuple(q.shape) == (R, K)


def test_rounding_of_ties_extremes_and_non_finite_blocks():
    from sln_amodal_amd import ops
    rows = []
    ties = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7.99])
    for e in (-126, -100, -20, 0, 30, 120, 124):             # top = 7.99 2^e: up to the largest float32 binades
        t = np.concatenate([ties, -ties]) * 2.0 ** e
        rows += [t, np.nextafter(t.astype(np.float32), np.float32(np.inf)).astype(np.float64),
                 np.nextafter(t.astype(np.float32), np.float32(-np.inf)).astype(np.float64)]
    for bad in (np.inf, -np.inf, np.nan):
        t = np.ones(32)
        t[31] = bad
        rows.append(t)
    rows += [np.zeros(32), -np.zeros(32), np.full(32, 2.0 ** -149), np.full(32, 2.0 ** -127), np.full(32, 3.4e38)]
    x = torch.from_numpy(np.stack(rows).astype(np.float32))
    q = ops.mx4_quantize(x.cuda())
    v = _check_codes(q, x)
    assert torch.equal(torch.nan_to_num(q.dequantize().cpu(), nan=777.0),
                       torch.nan_to_num(torch.from_numpy(v).float(), nan=777.0))


def test_rounding_reads_strided_rows_and_keeps_leading_axes():
    from sln_amodal_amd import ops
    base = _x((6, 100), 5).cuda()
    for view in (base[:, 3:70], base[::2, 1:], base.t(), base[:1].expand(4, 100), base.view(2, 3, 100)[:, 1:, :64],
                 base[:, :1], base[2]):
        q = ops.mx4_quantize(view)
        want = ops.mx4_quantize(view.contiguous())
        assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
        assert q.shape == view.shape and torch.equal(q.dequantize().cpu().double(),
                                                     ref.values(view.reshape(-1, view.shape[-1])).view(view.shape))
    assert ops.mx4_quantize(base[:0]).dequantize().shape == (0, 100)


def _product_bound(xq, wq, y, scale, bias, dtype):
    K = xq.shape[1]
    mag = xq.abs() @ wq.abs().t()
    if scale is not None:
        mag = mag * scale.double().abs()
    if bias is not None:
        mag = mag + bias.double().abs()
    # K additions of the sum, one rounding each for scale and bias, one to the type; fp16's subnormals: 2^-25
    return (K + 3) * 2.0 ** -23 * mag + torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * y.abs() + 2.0 ** -25


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,relu,affine", [
    (1, 1, 1, False, False), (1, 1024, 12544, True, True), (13, 324, 1024, False, True), (16, 17, 33, True, False),
    (17, 16, 255, False, True), (128, 128, 256, False, False), (129, 127, 257, True, True), (37, 1024, 1000, False, True),
    (1000, 81, 3000, True, True), (300, 300, 64, False, False),
    (6201, 2001, 70, True, True), (6145, 1793, 300, False, False)])      # (the large tiles)
def test_product_matches_the_definition(M, N, K, relu, affine, dtype):
    from sln_amodal_amd import ops
    x, w = _x((M, K), M + K, dtype), _x((N, K), N * 7 + K) / K ** 0.5
    g = torch.Generator().manual_seed(3)
    scale = torch.exp(0.3 * torch.randn(N, generator=g)) if affine else None
    bias = torch.randn(N, generator=g) if affine else None
    c = lambda t: None if t is None else t.cuda()
    xv, wv = ref.values(x), ref.values(w)
    y = xv @ wv.t()
    if affine:
        y = y * scale.double() + bias.double()
    bound = _product_bound(xv, wv, y, scale, bias, dtype)
    y = y.clamp(min=0) if relu else y
    wq = ops.mx4_quantize(w.cuda())
    got = ops.mx4_linear(x.cuda(), wq, c(bias), scale=c(scale), relu=relu)
    assert got.dtype == dtype and tuple(got.shape) == (M, N)
    assert ((got.cpu().double() - y).abs() <= bound).all()
    # the weight rounded in the call is the same weight; a second call gives the same bits
    assert torch.equal(got, ops.mx4_linear(x.cuda(), w.cuda(), c(bias), scale=c(scale), relu=relu))


@pytest.mark.parametrize("M", [1, 2, 16, 17, 64, 200, 520])
@pytest.mark.parametrize("K", [32, 320, 2304])
def test_sums_that_float32_holds_are_exact(M, K):
    """Levels under one scale: every partial sum is a multiple of 1/4 below 2^22, any order is exact.  Every block gets its
    own scale 2^0 or 2^1 by its largest level."""
    from sln_amodal_amd import ops
    g = torch.Generator().manual_seed(M + K)
    lev = torch.tensor(ref.LEVELS, dtype=torch.float32)
    N = 150
    x = lev[torch.randint(0, 8, (M, K), generator=g)] * (1 - 2 * torch.randint(0, 2, (M, K), generator=g))
    w = lev[torch.randint(0, 8, (N, K), generator=g)] * (1 - 2 * torch.randint(0, 2, (N, K), generator=g))
    x[:, ::32], w[:, ::32] = 6.0, -4.0
    x[:, 32::64] *= 1.0
    assert torch.equal(ref.values(x).float(), x)
    got = ops.mx4_linear(x.cuda(), w.cuda())
    assert torch.equal(got.cpu().double(), x.double() @ w.double().t())
    gy = torch.randint(-8, 9, (M, N), generator=g).float()
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    b = torch.zeros(N, device="cuda", requires_grad=True)
    gx, gw, gb = torch.autograd.grad(ops.mx4_linear(xd, wd, b), (xd, wd, b), gy.cuda())
    assert torch.equal(gx.cpu().double(), gy.double() @ w.double())
    assert torch.equal(gw.cpu().double(), gy.double().t() @ x.double())
    assert torch.equal(gb.cpu(), gy.sum(0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,relu,affine", [
    (1, 1, 1, False, False), (3, 5, 40, True, True), (16, 324, 100, False, True), (65, 63, 257, True, True),
    (130, 129, 300, False, False), (501, 324, 1000, True, True), (1600, 6, 33, False, True),
    (301, 701, 12544, False, True), (2000, 33, 6400, True, False)])       # (the large tiles)
def test_gradients_match_the_straight_through_formula(M, N, K, relu, affine, dtype):
    from sln_amodal_amd import ops
    x, w = _x((M, K), M + K, dtype), _x((N, K), N * 7 + K) / K ** 0.5
    g = torch.Generator().manual_seed(9)
    scale = torch.exp(0.3 * torch.randn(N, generator=g)) if affine else None
    bias = 0.1 * torch.randn(N, generator=g)
    gy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    xd, wd, bd = x.cuda().requires_grad_(), w.cuda().requires_grad_(), bias.cuda().requires_grad_()
    sd = None if scale is None else scale.cuda()
    y = ops.mx4_linear(xd, wd, bd, scale=sd, relu=relu)
    gx, gw, gb = torch.autograd.grad(y, (xd, wd, bd), gy.cuda())
    xv, wv = ref.values(x), ref.values(w)
    z = gy.double()
    if relu:                       # the mask is the forward's own output: no value near zero decides differently
        z = torch.where(y.detach().cpu().double() > 0, z, torch.zeros_like(z))
    s = scale.double() if affine else torch.ones(N, dtype=torch.float64)
    want_x, want_w, want_b = (z * s) @ wv, (z * s).t() @ xv, z.sum(0)
    # z * scale: one rounding (float32) or cut to 16 bits (2^-15); then at most 3 additions per term
    cut = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -15
    bx = ((3 * N + 2) * 2.0 ** -23 + cut) * ((z * s).abs() @ wv.abs()) + \
        torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * want_x.abs() + 2.0 ** -25
    bw = (3 * M + 3) * 2.0 ** -23 * ((z * s).abs().t() @ xv.abs()) + 1e-30
    bb = (M + 2) * 2.0 ** -23 * z.abs().sum(0) + 1e-30
    assert gx.dtype == dtype and gw.dtype == gb.dtype == torch.float32
    assert ((gx.cpu().double() - want_x).abs() <= bx).all()
    assert ((gw.cpu().double() - want_w).abs() <= bw).all()
    assert ((gb.cpu().double() - want_b).abs() <= bb).all()
    # one gradient at a time, and twice: the same bits
    for i, want in enumerate((gx, gw, gb)):
        leaf = (xd, wd, bd)[i]
        args = [t if j == i else t.detach() for j, t in enumerate((xd, wd, bd))]
        y1 = ops.mx4_linear(args[0], args[1], args[2], scale=sd, relu=relu)
        assert torch.equal(y1, y) or (i != 1 and M <= 16)       # (few rows without a weight gradient: another order)
        if torch.equal(y1, y):
            assert torch.equal(torch.autograd.grad(y1, leaf, gy.cuda())[0], want)


def test_gradient_of_the_smooth_part_against_differences():
    """x enters through its rounded values: moving w^ by a multiple of its own codes (a power of two keeps the rounding)
    moves the output linearly, so <gy, dy> = <gw, dw> for dw = w and <gy, dy> = <gx, dx> for dx = x rounded."""
    from sln_amodal_amd import ops
    x, w = _x((40, 96), 1), _x((24, 96), 2)
    xv, wv = ref.values(x).float(), ref.values(w).float()
    gy = _x((40, 24), 3)
    xd, wd = xv.cuda().requires_grad_(), wv.cuda().requires_grad_()
    y = ops.mx4_linear(xd, wd)
    gx, gw = torch.autograd.grad(y, (xd, wd), gy.cuda())
    y2 = ops.mx4_linear(xv.cuda(), (2 * wv).cuda())            # values double exactly
    want = (gy.double() * (y2 - y.detach()).cpu().double()).sum().item()
    got = (gw.cpu().double() * wv.double()).sum().item()
    other = (gx.cpu().double() * xv.double()).sum().item()
    mag = (gy.double().abs() * (xv.double().abs() @ wv.double().abs().t())).sum().item()
    assert abs(got - want) <= 300 * 2.0 ** -23 * mag and abs(other - want) <= 300 * 2.0 ** -23 * mag


def test_non_finite_values_stay_where_they_belong():
    from sln_amodal_amd import ops
    x, w = _x((40, 96), 1), _x((24, 96), 2)
    x[3, 40] = float("inf")
    x[7, 0] = float("nan")
    w[5, 95] = float("-inf")
    for rows in (slice(0, 8), slice(0, 40)):
        y = ops.mx4_linear(x[rows].cuda(), w.cuda(), relu=True).cpu()
        bad = torch.zeros(y.shape, dtype=torch.bool)
        bad[3], bad[7], bad[:, 5] = True, True, True
        assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    # an infinite gradient entry reaches its own row of gx and its own row of gw, nothing else
    xg, wg = _x((40, 96), 1).cuda().requires_grad_(), _x((24, 96), 2).cuda().requires_grad_()
    gy = torch.ones(40, 24, device="cuda")
    gy[11, 6] = float("inf")
    gx, gw = torch.autograd.grad(ops.mx4_linear(xg, wg), (xg, wg), gy)
    assert not torch.isfinite(gx[11]).all() and torch.isfinite(gx[[i for i in range(40) if i != 11]]).all()
    assert not torch.isfinite(gw[6]).all() and torch.isfinite(gw[[i for i in range(24) if i != 6]]).all()


def test_empty_batches_strided_gradients_and_leading_axes():
    from sln_amodal_amd import ops
    w = _x((24, 96), 2).cuda().requires_grad_()
    b = torch.zeros(24, device="cuda", requires_grad=True)
    x0 = torch.zeros(0, 96, device="cuda", requires_grad=True)
    y = ops.mx4_linear(x0, w, b)
    assert tuple(y.shape) == (0, 24)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x0, w, b))
    assert gx.shape == x0.shape and not gw.any() and not gb.any()
    x = _x((2, 3, 5, 96), 4).cuda().requires_grad_()
    y = ops.mx4_linear(x, w, b)
    assert tuple(y.shape) == (2, 3, 5, 24)
    flat = ops.mx4_linear(x.reshape(30, 96), w, b)
    assert torch.equal(y.reshape(30, 24), flat)
    gy = torch.randn(24, 30, device="cuda").t()                 # column-major gradient
    a = torch.autograd.grad(flat, (x, w, b), gy, retain_graph=True)
    c = torch.autograd.grad(flat, (x, w, b), gy.contiguous(), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    one = torch.autograd.grad(flat.sum(), (x, w, b), retain_graph=True)      # an expanded gradient of ones
    two = torch.autograd.grad(flat, (x, w, b), torch.ones(30, 24, device="cuda"))
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_wrong_calls_are_refused():
    from sln_amodal_amd import ops
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
    wq = ops.mx4_quantize(w)
    bad = [(TypeError, dict(x=x.double(), weight=w)), (TypeError, dict(x=x, weight=w.half())),
           (ValueError, dict(x=x[:, :32], weight=w)), (ValueError, dict(x=x, weight=w[0])),
           (ValueError, dict(x=x, weight=wq, bias=torch.zeros(7, device="cuda"))),
           (TypeError, dict(x=x, weight=wq, bias=torch.zeros(8, device="cuda").half())),
           (ValueError, dict(x=x, weight=wq, bias=torch.zeros(8))),
           (RuntimeError, dict(x=x, weight=wq, scale=torch.ones(8, device="cuda", requires_grad=True))),
           (ValueError, dict(x=x[:, :0], weight=w[:, :0])), (RuntimeError, dict(x=x.cpu(), weight=w))]
    for err, kw in bad:
        with pytest.raises(err):
            ops.mx4_linear(**kw)
    with pytest.raises(ValueError):
        ops.mx4_quantize(torch.zeros(3, 0, device="cuda"))
    with pytest.raises(TypeError):
        ops.mx4_quantize(torch.zeros(3, 3, device="cuda", dtype=torch.int32))
    with pytest.raises(TypeError):
        wq.dequantize(torch.int8)
    y = ops.mx4_linear(x.requires_grad_(), w)
    g = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):                           # no second derivative
        torch.autograd.grad(g.sum(), x)


def test_side_streams_and_captured_graphs():
    from sln_amodal_amd import ops
    w = _x((324, 1000), 2).cuda()
    wq = ops.mx4_quantize(w)
    xs = [_x((m, 1000), m).cuda() for m in (3, 200)]
    want = [ops.mx4_linear(x, wq, relu=True) for x in xs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.mx4_linear(x, wq, relu=True) for x in xs]
        graphs, outs = [], []
        for x in xs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.mx4_linear(x, wq, relu=True))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for r in range(3):                                          # both graphs in turn, eager work between the replays
        for x in xs:
            x.copy_(_x(tuple(x.shape), 100 + r).cuda())
        eager = [ops.mx4_linear(x, wq, relu=True) for x in xs]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


@pytest.mark.parametrize("M,N,K", [(7, 20, 70), (300, 130, 1000)])
def test_a_captured_training_pass_replays(M, N, K):
    """Forward and backward in one graph (all of it on the stream that captures): every replay equals the eager pass over
    the same values, with eager passes of other tensors between the replays."""
    from sln_amodal_amd import ops

    def fresh(seed):
        return [_x((M, K), seed).cuda(), _x((N, K), seed + 1).cuda(), _x((N,), seed + 2).cuda(), _x((M, N), seed + 3).cuda()]

    def run(x, w, b, gy):
        y = ops.mx4_linear(x, w, b, relu=True)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), gy)

    static = fresh(1)
    for t in static[:3]:
        t.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(*static)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = run(*static)
    torch.cuda.current_stream().wait_stream(s)
    for r in range(3):
        new = fresh(10 * r + 20)
        with torch.no_grad():
            for t, v in zip(static, new):
                t.copy_(v)
        for t in new[:3]:
            t.requires_grad_(True)
        want = run(*new)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
