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
