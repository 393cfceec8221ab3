"""What the ``Dropout`` module gives in evaluation mode and at p = 0: the type
and the rounding of training, and no draw."""

import itertools

import pytest
import torch

import complex_conv2d as cc

BF, FP, HF = torch.bfloat16, torch.float32, torch.float16
PAIRS = [(FP, FP), (FP, BF), (FP, HF), (BF, BF), (BF, FP), (HF, HF), (HF, FP)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("xt, rt", PAIRS)
@pytest.mark.parametrize("p, training", [(0.5, False), (0.0, True)])
def test_type_and_rounding(p, training, xt, rt, device):
    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn(200, generator=gen).to(device, t) for t in (xt, rt))
    d = cc.Dropout(p, seed=3).train(training)
    y = d(x, residual=r)
    assert y.dtype == rt and torch.equal(y, (x.float() + r.float()).to(rt))
    assert d(x) is x and d.calls == 0


@pytest.mark.gpu
@pytest.mark.parametrize("xt, rt", PAIRS)
def test_same_type_as_in_training(xt, rt):
    x, r = torch.randn(64, device="cuda:0").to(xt), torch.randn(64, device="cuda:0").to(rt)
    d = cc.Dropout(0.5, seed=3)
    assert d(x, residual=r).dtype == d.eval()(x, residual=r).dtype


def test_gradients_in_evaluation_mode():
    for xt, rt in itertools.product((FP, BF), (FP, BF)):
        x, r = torch.ones(4, dtype=xt, requires_grad=True), torch.ones(4, dtype=rt, requires_grad=True)
        cc.Dropout(0.5).eval()(x, residual=r).sum().backward()
        assert x.grad.dtype == xt and r.grad.dtype == rt
        assert (x.grad == 1).all() and (r.grad == 1).all()
