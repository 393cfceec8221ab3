"""Counter-based dropout against the generator restated in Python."""

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, HF = torch.bfloat16, torch.float32, torch.float16


def _x(n, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(n, generator=g, device=DEV).to(dtype)


def _check(x, p, seed, offset, residual=None):
    y = cc.dropout(x, p, seed, offset, residual=residual)
    want, keep = ref.dropout(x, p, seed, offset, residual)
    mag = want.abs() if residual is None else want.abs() + residual.double().abs()
    # x, its scale (itself rounded), the sum: three float32 roundings.
    ref.assert_bounded(y, want, mag + x.double().abs() * 2, 3, "y")
    if residual is None:
        assert torch.equal(y != 0, keep & (x != 0))
    return y


@pytest.mark.parametrize("xt, rt", [(FP, None), (BF, None), (HF, None), (FP, FP), (FP, BF),
                                    (FP, HF), (BF, BF), (BF, FP), (HF, HF), (HF, FP)])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 4099])
def test_types_and_lengths(n, xt, rt):
    _check(_x(n, xt), 0.3, 12345678901234567, 7, None if rt is None else _x(n, rt, 1))


@pytest.mark.parametrize("seed, offset", [(0, 0), (-1, -1), (1 << 63, 1 << 40),
                                          ((1 << 32) - 1, (1 << 32) - 1), (1 << 32, 1 << 32)])
def test_seeds_and_offsets(seed, offset):
    _check(_x(515, FP), 0.5, seed, offset)


@pytest.mark.parametrize("p", [0.0, 1e-6, 1 / 65536, 0.1, 0.999, 0.99999, 1.0])
def test_probabilities(p):
    x = _x(3001, FP)
    y = _check(x, p, 5, 6)
    if p == 0.0:
        assert torch.equal(y, x)
    if p == 1.0:
        assert not y.any()


def test_dropped_special_values_are_zero():
    x = _x(4096, FP)
    _, keep = ref.dropout(x, 0.5, 9, 9)
    x[~keep] = float("nan")
    assert torch.equal(cc.dropout(x, 0.5, 9, 9) != 0, keep)
    x[~keep] = float("inf")
    r = torch.ones_like(x)
    assert torch.equal(cc.dropout(x, 0.5, 9, 9, residual=r)[~keep], r[~keep])


def test_kept_share_and_independence():
    """Share kept within 5 standard deviations; masks of two offsets agree as
    often as chance has it."""
    n, p = 1 << 22, 0.25
    x = torch.ones(n, device=DEV)
    a, b = cc.dropout(x, p, 1, 0) != 0, cc.dropout(x, p, 1, 1) != 0
    sd = (p * (1 - p) / n) ** 0.5
    assert abs(a.double().mean().item() - (1 - p)) < 5 * sd
    same = (1 - p) ** 2 + p ** 2
    assert abs((a == b).double().mean().item() - same) < 5 * (same * (1 - same) / n) ** 0.5


def test_long_tensor_reaches_high_counters():
    """Elements past 2^31: the last ones carry the mask of their own index."""
    n = (1 << 31) + 4099
    x = torch.ones(n, device=DEV, dtype=BF)
    y = cc.dropout(x, 0.5, 77, 3)
    first = n - 4099
    keep = torch.from_numpy(ref.parts(77, 3, first, 4099) >= ref.threshold(0.5)).to(DEV)
    assert torch.equal(y[first:] != 0, keep)


@pytest.mark.parametrize("start", [0, 1, 3])
def test_views(start):
    big = _x(8192, BF)
    _check(big[start:start + 4001], 0.2, 1, 2, _x(8192, FP, 2)[start + 1:start + 4002])
    x = _x(64 * 40, FP).view(64, 40).t()
    assert torch.equal(cc.dropout(x, 0.4, 3, 4), cc.dropout(x.contiguous(), 0.4, 3, 4))


def test_backward_is_the_same_mask():
    x, r, dy = _x(3003, BF), _x(3003, FP, 1), _x(3003, FP, 2)
    x.requires_grad_(), r.requires_grad_()
    cc.dropout(x, 0.3, 11, 12, residual=r).backward(dy)
    assert torch.equal(x.grad, cc.dropout(dy, 0.3, 11, 12).to(BF))
    assert torch.equal(r.grad, dy)


def test_offset_on_the_device_and_captured_graph():
    x = _x(5000, FP)
    off = torch.tensor([3], device=DEV, dtype=torch.int64)
    assert torch.equal(cc.dropout(x, 0.5, 8, off), cc.dropout(x, 0.5, 8, 3))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cc.dropout(x, 0.5, 8, off)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = cc.dropout(x, 0.5, 8, off)
        off.add_(1)
    for k in (3, 4, 5):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, cc.dropout(x, 0.5, 8, k))
    # The backward pass keeps the offset the forward saw.
    x.requires_grad_()
    off.fill_(21)
    out = cc.dropout(x, 0.5, 8, off)
    off.fill_(99)
    out.backward(torch.ones_like(out))
    assert torch.equal(x.grad, cc.dropout(torch.ones_like(x), 0.5, 8, 21))


def test_module():
    d = cc.Dropout(0.5, seed=4)
    x = _x(1000, FP)
    a, b = d(x), d(x, residual=x)
    assert torch.equal(a, cc.dropout(x, 0.5, 4, 0))
    assert torch.equal(b, cc.dropout(x, 0.5, 4, 1, residual=x))
    assert torch.equal(d.eval()(x), x)


def test_refusals():
    x = _x(16, FP)
    with pytest.raises(ValueError, match="p must"):
        cc.dropout(x, 1.1, 0)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        cc.dropout(x.double(), 0.5, 0)
    with pytest.raises(ValueError, match="shape"):
        cc.dropout(x, 0.5, 0, residual=x[:8])
    with pytest.raises(TypeError, match="16-bit input's type"):
        cc.dropout(x.bfloat16(), 0.5, 0, residual=x.half())
    with pytest.raises(TypeError, match="int64"):
        cc.dropout(x, 0.5, 0, torch.zeros(1, device=DEV))
