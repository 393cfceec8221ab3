"""The operators together: the example's block (convolution planes, layer
norm, gated feed-forward, dropout with residual) against the same formula in
64 bits, and a few training steps."""

import os
import sys

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(cc.__file__))),
                                "examples"))

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _block():
    from conv_token_block import ConvTokenBlock
    torch.manual_seed(3)
    block = ConvTokenBlock(16, 24, 96, p=0.25, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    planes = [torch.randn(2, 9, 11, 16, generator=g, device=DEV) for _ in range(2)]
    return block, planes


def test_block_matches_the_formula():
    """From the convolution's own planes on: the branch is off by the rounding
    of the normalised rows and of the hidden values (relative rms u / sqrt(3)
    each) and of its own result; the residual is exact."""
    block, planes = _block()
    with torch.no_grad():
        out = block(*planes)
        t = torch.cat(block.conv.forward_planar(*planes), dim=-1)
    rows = t.reshape(-1, 48)
    n = ref.norm(rows, block.norm.weight, block.norm.bias, block.norm.eps)[0]
    y, _ = ref.ffn(n, block.ffn.w_gate, block.ffn.w_up, block.ffn.w_down, "gelu")
    _, keep = ref.dropout(torch.ones_like(rows), 0.25, 1, 0)
    branch = out.reshape(-1, 48).double() - rows.double()
    assert not branch[~keep].any()
    want = y * 65536 / (65536 - ref.threshold(0.25))
    err = (branch - want)[keep].square().mean().sqrt() / want[keep].square().mean().sqrt()
    u = ref.ROUNDOFF[torch.bfloat16]
    # Rounded normalised rows enter twice (gate and up): 4 + 1 + 1 units of
    # u^2 / 3 together, twice that allowed.
    assert err <= 2 * u * (6 / 3) ** 0.5


def test_dropout_masks_change_from_call_to_call_and_stop_in_evaluation():
    block, planes = _block()
    with torch.no_grad():
        a, b = block(*planes), block(*planes)
        block.eval()
        c, d = block(*planes), block(*planes)
    assert not torch.equal(a, b) and torch.equal(c, d)


def test_gradients_reach_every_parameter_and_training_converges():
    from conv_token_block import train
    block, planes = _block()
    block(*planes).square().mean().backward()
    for name, p in block.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    losses = train(steps=30, batch=2, channels=16, size=12, hidden=64)
    assert losses[-1] < 0.5 * losses[0]
