"""Forward-mode derivatives: ``ComplexConv2d`` has none, and refuses a dual
tensor instead of dropping its tangent."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("planar", [False, True])
@pytest.mark.parametrize("grad", [False, True], ids=["frozen", "trained"])
def test_convolution_refuses_dual_tensors(grad, planar):
    conv = cc.ComplexConv2d(4, 4, 3, padding=1, device=DEV)
    conv.weight_real.requires_grad_(grad)
    if planar:
        args = tuple(torch.randn(1, 5, 5, 4, device=DEV) for _ in range(2))
        f = conv.forward_planar
    else:
        args = (torch.randn(1, 4, 5, 5, device=DEV, dtype=torch.complex64),)
        f = conv
    with fwd.dual_level():
        dual = [fwd.make_dual(t, torch.ones_like(t)) for t in args[-1:]]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*args[:-1], *dual)
        f(*args)


@pytest.mark.parametrize("planar", [False, True])
def test_gradient_of_a_dual_tensor_is_refused(planar):
    conv = cc.ComplexConv2d(4, 4, 3, padding=1, device=DEV)
    if planar:
        x = torch.randn(1, 5, 5, 4, device=DEV, requires_grad=True)
        y = conv.forward_planar(x, x.detach())[0]
    else:
        x = torch.randn(1, 4, 5, 5, device=DEV, dtype=torch.complex64, requires_grad=True)
        y = conv(x)
    with fwd.dual_level():
        dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)
