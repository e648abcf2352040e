"""What autograd and modules promise, kept by MLP's operator path."""
import pytest
import torch
from torch.autograd import forward_ad

from ivae_amd import MLP

pytestmark = pytest.mark.gpu
OPTS = [dict(layer_norm=True), dict(residual=True), dict(layer_norm=True, residual=True, dropout=.25)]


def mlp(seed=0, **opts):
    torch.manual_seed(seed)
    return MLP(12, 5, 40, 4, activation="gelu", **opts).cuda()


@pytest.mark.parametrize("opts", OPTS)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(opts, grad):
    """The kernels have no tangents: a dual input, or a dual parameter, is refused with gradients and without, never dropped."""
    m, x = mlp(**opts).eval(), torch.randn(7, 12, device="cuda")
    with torch.set_grad_enabled(grad):
        with forward_ad.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                m(forward_ad.make_dual(x, torch.ones_like(x)))
            w = m.fc[1].weight
            del m.fc[1].weight
            m.fc[1].weight = forward_ad.make_dual(w.detach(), torch.ones_like(w))
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                m(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(mlp(**opts).eval(), (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("opts", OPTS)
def test_without_gradients_nothing_is_kept(opts):
    m, x = mlp(**opts).eval(), torch.randn(2048, 12, device="cuda")
    y = m(x)
    assert y.grad_fn is not None
    with torch.no_grad():
        z = m(x)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        z = m(x)
        assert torch.cuda.memory_allocated() == before and z.grad_fn is None and torch.equal(z, y)
    with torch.inference_mode():
        assert torch.equal(m(x), y)


@pytest.mark.parametrize("opts", OPTS)
@pytest.mark.parametrize("grad", [True, False])
def test_tracing_records_the_operators_or_refuses(opts, grad):
    """A traced MLP computes what the MLP does on other inputs than the traced one; where it cannot, tracing is refused."""
    m = mlp(**opts).eval()
    x, other = torch.randn(7, 12, device="cuda"), torch.randn(7, 12, device="cuda")
    with torch.set_grad_enabled(grad):
        try:
            t = torch.jit.trace(m, x, check_trace=False)
        except RuntimeError as e:
            assert "trac" in str(e)
            return
        assert torch.equal(t(other), m(other))


def test_tracing_with_dropout_is_refused():
    m, x = mlp(**OPTS[-1]).train(), torch.randn(7, 12, device="cuda")
    with pytest.raises(RuntimeError, match="mask"):
        torch.jit.trace(m, x, check_trace=False)
