"""Layer norm on many rows of odd and of even width, so that a thread group
walks several: the ring's stages are used again, the shift of a group's rows
must not change, and the last row ends in a stage used before.  And odd rows
of more than 8192 features that are not dense."""

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc
from test_token_norm_gpu import BF, DEV, EPS, FP, HF, _check_backward, _check_forward, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(BF, FP, BF), (BF, BF, FP), (HF, HF, HF), (FP, FP, FP),
                                   (FP, FP, BF)], ids=lambda t: "-".join(str(d)[6:] for d in t))
@pytest.mark.parametrize("rows, features", [(12545, 1001), (5000, 7), (20011, 31), (20011, 33),
                                            (5000, 999), (3001, 4097), (5000, 250), (12545, 1002)])
def test_many_rows(rows, features, types):
    x, w, b, dy = _inputs(rows, features, types, seed=rows + features)
    mean, rstd = _check_forward(x, w, b, types[2])
    first = _check_backward(dy, x, mean, rstd, w)
    again = cc.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(a, c) for a, c in zip(first, again))


@pytest.mark.parametrize("rows", [300, 2500])
@pytest.mark.parametrize("features", [7, 33, 1001])
def test_special_values_stay_in_their_row(features, rows):
    """NaN and infinities in a neighbour that a shifted vector reads too."""
    x, w, b, dy = _inputs(rows, features, (BF, FP, BF))
    clean, mean, rstd = cc.layer_norm_with_stats(x, w, b, EPS)
    dx = cc.layer_norm_backward(dy, x, mean, rstd, w)[0]
    x[1::3] = float("nan")
    x[2::6] = float("inf")
    y, m, r = cc.layer_norm_with_stats(x, w, b, EPS)
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[1::3] = keep[2::6] = False
    assert torch.equal(y[keep], clean[keep]) and y[1::3].isnan().all()
    assert torch.equal(cc.layer_norm_backward(dy, x, m, r, w)[0][keep], dx[keep])


@pytest.mark.parametrize("types", [(BF, FP, BF), (FP, FP, FP)], ids=["bf16", "f32"])
@pytest.mark.parametrize("features", [8193, 16383, 20001, 33001])
def test_wide_rows_with_gaps(features, types):
    x, w, b, dy = _inputs(9, features + 6, types, seed=features)
    x, dy, w, b = x[:, 3:-3], dy[:, 1:-5], w[2:-4], b[:-6]
    mean, rstd = _check_forward(x, w, b, types[2])
    _check_backward(dy, x, mean, rstd, w)
