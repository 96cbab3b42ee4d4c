"""Forward-mode differentiation is refused where a kernel would drop the tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused():
    from sln_amodal_amd import ops
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(s, generator=g).cuda() for s in ((30, 64), (20, 64), (20,)))
    wq = ops.mx4_quantize(w)
    plain = ops.mx4_linear(x, w, b)
    ortho = ops.orthogonalize(w)
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))
        for args, kw in (((d(x), w, b), {}), ((x, d(w), b), {}), ((x, w, d(b)), {}), ((d(x), wq), {}), ((d(x[:3]), wq), {}),
                         ((x, w, b), dict(scale=d(b)))):
            with pytest.raises(RuntimeError):
                ops.mx4_linear(*args, **kw)
            with pytest.raises(RuntimeError), torch.no_grad():
                ops.mx4_linear(*args, **kw)
        for arg in (d(w), [w, d(x)]):
            with pytest.raises(RuntimeError):
                ops.orthogonalize(arg)
        assert torch.equal(ops.mx4_linear(x, w, b), plain) and torch.equal(ops.orthogonalize(w), ortho)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ops.mx4_linear(t, wq), (x,), (torch.ones_like(x),))
