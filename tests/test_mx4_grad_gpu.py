"""GPU tests of what the 4-bit layer's gradients owe: sums of float32 products whatever the gradients' type, every tile and
launch that the sizes can reach, and what a NaN does.  Tolerances as in test_mx4_gpu: n terms n 2^-23 of the sum of
magnitudes per addition, the result's own rounding eps / 2; where all sums are exactly representable the bits are equal."""
import pytest
import torch

from tests import _mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(3, 2, 32), (40, 16, 96), (200, 8, 320), (2100, 14, 6400)])
def test_a_scaled_gradient_keeps_what_cancellation_leaves(M, N, K, dtype):
    """z = +-1, scale = 1 + 2^-9 + j 2^-20, weights 1: every partial sum is a multiple of 2^-20 below 2^4, so float32 products
    and sums are exact, and what is left after the large bits cancel is what two bf16 parts of the scale do not hold."""
    from sln_amodal_amd import ops
    g = torch.Generator().manual_seed(M + N)
    scale = 1 + 2.0 ** -9 + torch.randint(0, 16, (N,), generator=g).float() * 2.0 ** -20
    sign = torch.ones(M, N)
    sign[:, 1::2] = -1
    x = torch.ones(M, K)
    w = torch.ones(N, K)
    assert torch.equal(ref.values(w).float(), w)
    xd = x.to(dtype).cuda().requires_grad_()
    wd = w.cuda().requires_grad_()
    y = ops.mx4_linear(xd, wd, scale=scale.cuda())
    gx, gw = torch.autograd.grad(y, (xd, wd), sign.to(dtype).cuda())
    want = ((sign.double() * scale.double()) @ w.double()).to(dtype)       # multiples of 2^-20 below 2^-15: exact in any type
    assert torch.equal(want.double(), (sign.double() * scale.double()) @ w.double())
    assert torch.equal(gx.cpu(), want)
    assert torch.equal(torch.autograd.grad(ops.mx4_linear(xd, wd.detach(), scale=scale.cuda()), xd, sign.to(dtype).cuda())[0], gx)
    # gw = scale sum(z): integers below 2^12 times scale, one rounding to float32
    assert torch.equal(gw.cpu(), (scale * sign.sum(0))[:, None].expand(N, K))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scaled_16_bit_gradients_are_as_near_as_float32_ones(dtype):
    """The 64-bit result rounded to the type, but where it lies within the float32 sums' bound of a border between two
    values: the terms' own roundings (2^-24) and N additions."""
    from sln_amodal_amd import ops
    M, N, K = 300, 324, 512
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(M, K, generator=g).to(dtype), torch.randn(N, K, generator=g) / K ** 0.5
    scale = torch.exp(0.2 * torch.randn(N, generator=g))
    gy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g)) * 1e-2).to(dtype)
    xd = x.cuda().requires_grad_()
    gx = torch.autograd.grad(ops.mx4_linear(xd, w.cuda(), scale=scale.cuda()), xd, gy.cuda())[0].cpu()
    wv, zs = ref.values(w), gy.double() * scale.double()
    want = zs @ wv
    slack = (3 * N + 3) * 2.0 ** -23 * (zs.abs() @ wv.abs())
    lo, hi = (want - slack).to(dtype), (want + slack).to(dtype)
    assert ((gx == lo) | (gx == hi) | ((gx > lo) & (gx < hi))).all()


def _large(rows, cols):
    """csrc/mx4_grad.hip (mg_large): 128 x 256 tiles from 384 of them on."""
    return (-(-rows // 128)) * (-(-cols // 256)) >= 384


@pytest.mark.parametrize("M,N,K,gx_large,gw_large", [(130, 1025, 11010, False, True), (1100, 1030, 10900, True, True),
                                                     (1100, 130, 10900, True, False)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_on_the_large_tiles(M, N, K, gx_large, gw_large, dtype):
    from sln_amodal_amd import ops
    assert (_large(M, K), _large(N, K)) == (gx_large, gw_large)
    g = torch.Generator().manual_seed(M + N)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g))).to(dtype)
    w = torch.randn(N, K, generator=g) / K ** 0.5
    scale, bias = torch.exp(0.3 * torch.randn(N, generator=g)), 0.1 * torch.randn(N, generator=g)
    gy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    xd, wd, bd = x.cuda().requires_grad_(), w.cuda().requires_grad_(), bias.cuda().requires_grad_()
    y = ops.mx4_linear(xd, wd, bd, scale=scale.cuda(), relu=True)
    gx, gw, gb = torch.autograd.grad(y, (xd, wd, bd), gy.cuda())
    # (the reference's products in 64 bits on the device: plain matrices, no batches)
    xv, wv, s = ref.values(x).cuda(), ref.values(w).cuda(), scale.double().cuda()
    z = torch.where(y.detach() > 0, gy.cuda().double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    zs = z * s
    want_x, mag_x = zs @ wv, zs.abs() @ wv.abs()
    zt = zs.t().contiguous()
    want_w, mag_w = zt @ xv, zt.abs() @ xv.abs()
    bx = ((3 * N + 2) * 2.0 ** -23 + 2.0 ** -24) * mag_x + torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * want_x.abs() + 2.0 ** -25
    assert ((gx.double() - want_x).abs() <= bx).all()
    assert ((gw.double() - want_w).abs() <= (3 * M + 3) * 2.0 ** -23 * mag_w + 1e-30).all()
    assert ((gb.double() - z.sum(0)).abs() <= (M + 2) * 2.0 ** -23 * z.abs().sum(0) + 1e-30).all()
    for i, want in enumerate((gx, gw, gb)):                        # one at a time: the same bits
        args = [t if j == i else t.detach() for j, t in enumerate((xd, wd, bd))]
        y1 = ops.mx4_linear(args[0], args[1], args[2], scale=scale.cuda(), relu=True)
        assert torch.equal(y1, y) and torch.equal(torch.autograd.grad(y1, (xd, wd, bd)[i], gy.cuda())[0], want)


@pytest.mark.parametrize("rows", [12, 40])
def test_relu_stops_the_gradient_where_the_output_is_nan(rows):
    """y > 0 is false for a NaN, as in the framework's convolutions (torch's relu lets the gradient through there): the bias
    counts the other rows only.  The NaN is not hidden: the weight's gradient meets it in x."""
    from sln_amodal_amd import ops
    g = torch.Generator().manual_seed(rows)
    x, w, b = torch.rand(rows, 64, generator=g), torch.rand(20, 64, generator=g), torch.zeros(20)
    x[3, 7] = float("nan")
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x, w, b))
    y = ops.mx4_linear(xd, wd, bd, relu=True)
    assert torch.isnan(y[3]).all() and (y[:3] > 0).all() and (y[4:] > 0).all()
    gx, gw, gb = torch.autograd.grad(y, (xd, wd, bd), torch.ones_like(y))
    assert torch.equal(gb.cpu(), torch.full((20,), float(rows - 1)))
    assert not gx[3].any() and torch.isfinite(gx).all()
    assert torch.isnan(gw[:, :32]).all() and torch.isfinite(gw[:, 32:]).all()


def test_more_rows_than_the_gradients_take_are_refused_before_the_forward():
    from sln_amodal_amd import ops
    w = torch.ones(3, 32, device="cuda")
    x = torch.ones(1, 32, device="cuda").expand((1 << 21) + 1, 32)
    assert torch.equal(ops.mx4_linear(x, w)[-1], torch.full((3,), 32.0, device="cuda"))
    with pytest.raises(ValueError):
        ops.mx4_linear(x, w.requires_grad_())
    with pytest.raises(ValueError):
        ops.mx4_linear(torch.ones(2, 1, device="cuda", requires_grad=True), torch.ones(1, 1, device="cuda").expand((1 << 21) + 1, 1))
    x = x[:-1]
    gx, gw = torch.autograd.grad(ops.mx4_linear(x.requires_grad_(), w).sum(), (x, w))
    assert (gx == 3).all() and (gw == 2.0 ** 21).all()
