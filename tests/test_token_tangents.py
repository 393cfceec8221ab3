"""Forward-mode derivatives: the operators have none, and refuse a dual tensor
instead of dropping its tangent."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def _calls():
    x = torch.randn(4, 16, device=DEV)
    w, b = torch.ones(16, device=DEV), torch.zeros(16, device=DEV)
    h, wg, wu = x.to(BF), torch.randn(24, 16, device=DEV).to(BF), torch.randn(24, 16, device=DEV).to(BF)
    wd = torch.randn(16, 24, device=DEV).to(BF)
    return {"layer_norm": (cc.layer_norm, (x, w, b)),
            "gated_feed_forward": (cc.gated_feed_forward, (h, wg, wu, wd)),
            "dropout": (lambda t, r: cc.dropout(t, 0.5, 1, residual=r), (x, x))}


@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("name", ["layer_norm", "gated_feed_forward", "dropout"])
def test_dual_tensors_are_refused(name, which, grad):
    f, args = _calls()[name]
    if which >= len(args):
        return
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = [fwd.make_dual(t, torch.ones_like(t)) if i == which else t
                for i, t in enumerate(args)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*dual)
        f(*args)  # tensors without a tangent pass


@pytest.mark.parametrize("name", ["layer_norm", "gated_feed_forward", "dropout"])
def test_jvp_is_refused(name):
    f, args = _calls()[name]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, args, tuple(torch.ones_like(t) for t in args))


@pytest.mark.parametrize("name", ["layer_norm", "gated_feed_forward", "dropout"])
def test_gradient_of_a_dual_tensor_is_refused(name):
    f, args = _calls()[name]
    x = args[0].requires_grad_()
    y = f(x, *args[1:])
    with fwd.dual_level():
        dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)
