"""GPU tests of the orthogonalisation at the ends of its range: norms next to and beyond float32's largest, every eps.
Tolerances as in test_ortho_gpu."""
import pytest
import torch

from tests import _mx4_ref as ref
from tests.test_ortho_gpu import _matrix, _rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(64, 576), (576, 64), (200, 210), (1000, 1000), (140, 2700), (2700, 140)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matrices_whose_norm_float32_does_not_hold(rows, cols, dtype):
    """Entries up to 2^127: the same as of the matrix times 2^-100 (exactly scaled; eps is nothing beside either norm)."""
    from sln_amodal_amd import ops
    g = _matrix(rows, cols, 3, 1.0)
    g = (g / g.abs().max()).to(dtype)
    small, large = g.float() * 2.0 ** 27, (g.float() * 2.0 ** 127).to(dtype)
    assert torch.isfinite(large).all() and large.double().norm() > 2.0 ** 128
    want = ref.orthogonal(small)
    tol = 8 * _rel(ref.orthogonal(small, dtype=torch.float32), want) + 2.0 ** -20
    tol += torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
    got = ops.orthogonalize([large.cuda(), small.to(dtype).cuda()])
    for o in got:
        assert _rel(o.cpu(), want) <= tol, _rel(o.cpu(), want)


def _iterate(x):
    for _ in range(5):
        a = x @ x.t()
        x = ref.NS[0] * x + (ref.NS[1] * a + ref.NS[2] * a @ a) @ x
    return x


@pytest.mark.parametrize("eps", [1e30, 1e-30])
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e30, 1e36])
@pytest.mark.parametrize("rows,cols", [(40, 90), (130, 300)])
def test_any_eps(rows, cols, size, eps):
    """The control starts from the float32 X: a float32 norm would overflow where the matrix does not."""
    from sln_amodal_amd import ops
    g = _matrix(rows, cols, 5, size)
    x = g.double() / (g.double().norm() + eps)
    want = _iterate(x).float()
    tol = 8 * _rel(_iterate(x.float()), want) + 2.0 ** -20
    got = ops.orthogonalize(g.cuda(), eps=eps).cpu()
    assert _rel(got, want) <= tol, (_rel(got, want), tol)


@pytest.mark.parametrize("rows,cols", [(64, 576), (500, 700), (140, 30000)])
@pytest.mark.parametrize("size", [1.0, 1.1, 1.9])
def test_powers_of_two_change_no_bit(rows, cols, size):
    """The norm is up to 2^139, where a float32 of 1 / norm has ten bits left."""
    from sln_amodal_amd import ops
    g = torch.sign(torch.randn(rows, cols, generator=torch.Generator().manual_seed(1))) * size
    assert torch.equal(ops.orthogonalize((g * 2.0 ** 127).cuda()), ops.orthogonalize((g * 2.0 ** 27).cuda()))
