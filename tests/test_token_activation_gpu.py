"""The activations and their slopes, element by element: weights that pick one
product per output make y = act(g), dx_0 = act'(g) and dx_1 = act(g) for one
hidden unit, over every 16-bit g in a range.

Bounds, besides the result's own rounding.  SiLU: two hardware approximations
(2^x, 1/x: 2 units of 2^-23 each) and the rounded exponent, relative
(|g| + 8) 2^-23.  GELU's distribution: 0.75e-7 from its series (Abramowitz and
Stegun 7.1.26) and six float32 roundings of values up to 1, absolute; times g.
Its slope adds g phi(g), whose exponent g^2/2 is rounded: relative
(g^2 + 8) 2^-23.  Where g is kept for the backward pass it has 15 bits after
the first: |g| 2^-15 more, times the derivative.  A result below the type's
normal numbers is rounded to a multiple of its smallest one."""

import math

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PHI = 0.75e-7 + 6 * 2.0 ** -24
# Half the smallest number of each type.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def _gates(dtype, most):
    """Every value of the type between -most and most, but subnormals."""
    v = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype).double()
    v = v[(v.abs() <= most) & (v.abs() >= torch.finfo(dtype).tiny)]
    return torch.cat((v.sort().values, torch.zeros(1, dtype=torch.double))).to(dtype).to(DEV)


def _exact(g, activation):
    """(value, slope, error of the value, error of the slope)."""
    g = g.double()
    if activation == "silu":
        s = torch.sigmoid(g)
        value, slope = g * s, s * (1 + g * (1 - s))
        rel = (g.abs() + 8) * 2.0 ** -23
        return value, slope, rel * value.abs(), rel * (s + value.abs() * s + value.abs())
    c, phi = torch.special.ndtr(g), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return (g * c, c + g * phi, g.abs() * PHI,
            PHI + g.abs() * phi * (g * g + 8) * 2.0 ** -23)


def _weights(dtype, hidden):
    wg = torch.zeros(hidden, 8, device=DEV, dtype=dtype)
    wu, wd = torch.zeros_like(wg), torch.zeros(8, hidden, device=DEV, dtype=dtype)
    wg[0, 0] = wu[0, 1] = wd[0, 0] = 1
    return wg, wu, wd


def _check(got, want, error, what):
    ref_error = ref.ROUNDOFF[got.dtype] * (want.abs() + error) + error + TINY[got.dtype]
    ratio = ((got.double() - want).abs() / ref_error.clamp_min(1e-300)).max().item()
    assert ratio <= 1, f"{what}: {ratio:.2f} x the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("hidden, repeat", [(8, 1), (128, 1), (128, 3)])
def test_values_and_slopes(hidden, repeat, activation, dtype):
    """Few tiles: the backward pass reads g; many (repeat): it computes g again."""
    g = _gates(dtype, 12.0).repeat(repeat)
    x = torch.zeros(g.numel(), 8, device=DEV, dtype=dtype)
    x[:, 0], x[:, 1] = g, 1
    w = _weights(dtype, hidden)
    value, slope, ev, es = _exact(g, activation)
    y, saved = cc.gated_feed_forward_with_saved(x, *w, activation)
    _check(y[:, 0], value, ev, "value")
    assert torch.equal(y, cc.gated_feed_forward(x, *w, activation)) and not y[:, 1:].any()
    dy = torch.zeros_like(x)
    dy[:, 0] = 1
    dx = cc.gated_feed_forward_backward(dy, saved, x, *w, activation)[0]
    kept = saved.shape[0] > 1
    assert kept == (repeat == 1)
    if kept:
        _, first, second = ref._act(g.double(), activation)
        es = es + 2.0 ** -15 * (g.double() * second).abs()
        ev = ev + 2.0 ** -15 * (g.double() * first).abs()
    _check(dx[:, 0], slope, es, "slope")
    _check(dx[:, 1], value, ev, "value in the gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_values_of_few_rows(activation, dtype):
    """The kernels for up to 16 rows."""
    g = _gates(dtype, 12.0)[::97]
    w = _weights(dtype, 64)
    for first in range(0, g.numel(), 13):
        part = g[first:first + 13]
        x = torch.zeros(part.numel(), 8, device=DEV, dtype=dtype)
        x[:, 0], x[:, 1] = part, 1
        value, _, ev, _ = _exact(part, activation)
        _check(cc.gated_feed_forward(x, *w, activation)[:, 0], value, ev, "value")
