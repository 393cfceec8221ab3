"""Gated feed-forward block where the backward pass computes the projections
again (up to 512 features and enough tiles for the GPU): both types and
activations, sizes that no vector divides, parts of the gradients."""

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc
from test_token_ffn_gpu import BF, HF, _check, _inputs

pytestmark = pytest.mark.gpu


def _assert_recomputes(x, wg, wu, wd):
    """One plane kept (h) instead of four."""
    assert cc.gated_feed_forward_with_saved(x, wg, wu, wd)[1].shape[0] == 1


@pytest.mark.parametrize("rows, features, hidden, dtype, activation", [
    (25088, 256, 1024, HF, "gelu"), (2200, 512, 2304, BF, "silu"), (2200, 512, 2304, HF, "silu"),
    (10000, 131, 517, BF, "gelu"), (10000, 131, 517, HF, "silu"), (9000, 77, 640, BF, "silu"),
    (9000, 128, 515, HF, "gelu"), (40001, 8, 16, BF, "gelu"), (38000, 1, 1, BF, "silu")])
def test_shapes_and_types(rows, features, hidden, dtype, activation):
    x, wg, wu, wd, dy = _inputs(rows, features, hidden, dtype, seed=rows)
    _assert_recomputes(x, wg, wu, wd)
    _check(x, wg, wu, wd, dy, activation)


@pytest.mark.parametrize("rows, features, hidden", [(5000, 328, 1032), (10000, 131, 517),
                                                    (9000, 128, 515)])
def test_parts_of_the_gradients(rows, features, hidden):
    """Bits may differ from the call for all of them (the last wave's split
    depends on the tiles): each against the definition."""
    x, wg, wu, wd, dy = _inputs(rows, features, hidden)
    _assert_recomputes(x, wg, wu, wd)
    want, rss = ref.ffn_backward(dy, x, wg, wu, wd, "silu")
    for need in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 1), (0, 1, 1, 0)):
        ts = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, wg, wu, wd), need)]
        cc.gated_feed_forward(*ts).backward(dy)
        for i, (t, n) in enumerate(zip(ts, need)):
            if n:
                ref.assert_product(t.grad, want[i], rss[i], str(need))
            else:
                assert t.grad is None


def test_strided_rows():
    big, wg, wu, wd, bigdy = _inputs(6000, 400, 1024)
    for offset in (0, 1, 8):
        x, dy = big[:, offset:offset + 136], bigdy[:, offset:offset + 136]
        ws = wg[:, :136].contiguous(), wu[:, :136].contiguous(), wd[:136].contiguous()
        _assert_recomputes(x, *ws)
        _check(x, *ws, dy, "gelu")
