"""Gradient of dropout where the branch and the residual differ in type: dx in
x's type from dy in the residual's, with the one rounding of its own type."""

import ctypes

import pytest
import torch

import ccv_abi
import token_reference as ref
import complex_conv2d as cc

DEV = "cuda:0"
BF, FP, HF = torch.bfloat16, torch.float32, torch.float16


def _gradient(x, residual, p, seed, offset, dy):
    x = x.detach().clone().requires_grad_()
    cc.dropout(x, p, seed, offset, residual=residual).backward(dy)
    return x.grad


@pytest.mark.gpu
@pytest.mark.parametrize("xt, rt", [(FP, BF), (FP, HF), (BF, FP), (HF, FP), (BF, BF), (FP, FP)])
@pytest.mark.parametrize("n", [1, 9, 8192, 40003])
def test_one_rounding(n, xt, rt):
    g = torch.Generator(device=DEV).manual_seed(n)
    x, r, dy = (torch.randn(n, generator=g, device=DEV).to(t) for t in (xt, rt, rt))
    dx = _gradient(x, r, 0.3, 5, 6, dy)
    assert dx.dtype == xt
    want, keep = ref.dropout(dy, 0.3, 5, 6)
    # The rounded scale and the product, in float32, then the result.
    ref.assert_bounded(dx, want, want.abs(), 2, "dx")
    assert torch.equal(dx != 0, keep & (dy != 0))


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.75, 1.0])
def test_float32_gradient_beyond_float16(p):
    """dy near float16's largest number, scaled past it."""
    dy = torch.full((64,), 60000.0, device=DEV, dtype=HF)
    dx = _gradient(torch.ones(64, device=DEV), torch.ones(64, device=DEV, dtype=HF), p, 1, 2, dy)
    want, _ = ref.dropout(dy, p, 1, 2)
    assert dx.dtype == FP and torch.equal(dx.double(), want)


@pytest.mark.gpu
def test_views_and_offset_on_the_device():
    big = torch.randn(5001, device=DEV)
    off = torch.tensor([9], device=DEV)
    x = torch.ones(1000, device=DEV, dtype=BF).requires_grad_()
    cc.dropout(x, 0.5, 3, off, residual=torch.zeros(1000, device=DEV)).backward(big[1:2001:2])
    want, _ = ref.dropout(big[1:2001:2], 0.5, 3, 9)
    ref.assert_bounded(x.grad, want, want.abs(), 2, "dx")


P, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)  # never dereferenced by the checks


def _call(dy=P, dyt=0, dx=P, dxt=1, count=8, p=0.5):
    ccv_abi.load()
    f = ctypes.CDLL(ccv_abi.LIB).ccv_dropout_backward
    f.restype = ctypes.c_int
    rc = f(dy, ctypes.c_int(dyt), dx, ctypes.c_int(dxt), ctypes.c_int64(count), ctypes.c_double(p),
           ctypes.c_uint64(1), ctypes.c_uint64(2), None, None)
    return rc, ccv_abi.last_error()


@pytest.mark.parametrize("kw, status, text", [
    (dict(p=-0.1), 1, "p must"), (dict(p=float("nan")), 1, "p must"), (dict(count=-1), 1, "count"),
    (dict(dyt=5), 1, "element type"), (dict(dxt=-1), 1, "element type"),
    (dict(dyt=1, dxt=2), 1, "16-bit"), (dict(dy=None), 1, "null"), (dict(dx=ODD), 1, "aligned"),
    (dict(count=1 << 50), 2, "too large"),
])
def test_refusals(kw, status, text):
    rc, msg = _call(**kw)
    assert rc == status and text in msg


def test_nothing_to_do_launches_nothing():
    assert _call(dy=None, dx=None, count=0)[0] == 0
