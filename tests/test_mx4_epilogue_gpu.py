"""act(sum * scale + bias) is rounded once after each operation, by every kernel that ends a 4-bit product: where the sums are
exactly representable, the results are those of elementary float32 operations, bit for bit."""
import pytest
import torch

from tests import _mx4_ref as ref

pytestmark = pytest.mark.gpu


# few rows (with and without cuts of the contraction), many (the same), the large tiles
@pytest.mark.parametrize("M,N,K", [(5, 40, 32), (16, 300, 2304), (17, 150, 320), (200, 150, 2304), (6201, 2001, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_exact_sums_are_scaled_and_shifted_in_single_roundings(M, N, K, dtype):
    from sln_amodal_amd import ops
    g = torch.Generator().manual_seed(M + K)
    lev = torch.tensor(ref.LEVELS, dtype=torch.float32)
    x = lev[torch.randint(0, 8, (M, K), generator=g)] * (1 - 2 * torch.randint(0, 2, (M, K), generator=g))
    w = lev[torch.randint(0, 8, (N, K), generator=g)] * (1 - 2 * torch.randint(0, 2, (N, K), generator=g))
    x[:, ::32], w[:, ::32] = 6.0, -4.0                      # one scale for all blocks: sums are multiples of 1/4 below 2^20
    scale = torch.exp(0.3 * torch.randn(N, generator=g)) * 0.01
    bias = torch.randn(N, generator=g)
    acc = (x.cuda().double() @ w.cuda().double().t().contiguous()).float()
    want = (acc * scale.cuda() + bias.cuda()).to(dtype)     # two launches: no fused multiply-add
    xd, sd, bd = x.to(dtype).cuda(), scale.cuda(), bias.cuda()
    for weight in (w.cuda(), ops.mx4_quantize(w.cuda())):
        assert torch.equal(ops.mx4_linear(xd, weight, bd, scale=sd), want)
        assert torch.equal(ops.mx4_linear(xd, weight, bd, scale=sd, relu=True), want.clamp(min=0))
        assert torch.equal(ops.mx4_linear(xd, weight, bd), (acc + bd).to(dtype))
        assert torch.equal(ops.mx4_linear(xd, weight, scale=sd), (acc * sd).to(dtype))
