"""mx.linear and mx.swiglu have no forward-mode derivative: a tangent is refused, whether or not a gradient is asked for."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

from mor_amd import mx


def empty(*shape, device="cuda"):
    return torch.empty(*shape, dtype=torch.bfloat16, device=device)


CALLS = [("linear, x", lambda x, w, d: mx.linear(d, w)), ("linear, 3-D x", lambda x, w, d: mx.linear(d.view(2, 32, 64), w)),
         ("linear, weight", lambda x, w, d: mx.linear(x, d)), ("swiglu, gate", lambda x, w, d: mx.swiglu(d, x)),
         ("swiglu, up", lambda x, w, d: mx.swiglu(x, d)), ("swiglu, 3-D", lambda x, w, d: mx.swiglu(d.view(2, 32, 64), d.view(2, 32, 64)))]


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c[0])
@pytest.mark.parametrize("gradients", [True, False])
def test_dual_tensors_are_refused(call, gradients):
    with FakeTensorMode(), forward_ad.dual_level():
        x, w = empty(64, 64), empty(32, 64)
        dual = forward_ad.make_dual(empty(64, 64), empty(64, 64))
        with torch.set_grad_enabled(gradients), pytest.raises(RuntimeError, match="forward-mode"):
            call[1](x, w, dual)
        call[1](x, w, forward_ad.unpack_dual(dual).primal)         # without its tangent


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c[0])
def test_jvp_is_refused(call):
    with FakeTensorMode():
        x, w, t = empty(64, 64), empty(32, 64), empty(64, 64)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(lambda d: call[1](x, w, d), (empty(64, 64),), (t,))


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_tangents_of_the_gradient_are_refused():
    x, w = empty(64, 64).zero_().requires_grad_(), empty(32, 64).zero_().requires_grad_()
    for y in (mx.linear(x, w), mx.swiglu(x, x)):
        dy = torch.ones_like(y)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, x, forward_ad.make_dual(dy, dy), retain_graph=True)
        assert torch.autograd.grad(y, x, dy)[0].shape == x.shape
