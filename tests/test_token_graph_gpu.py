"""The operators in a captured graph: replays give the eager results, on new
inputs too."""

import pytest
import torch

import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# One row, a ragged few hundred, sizes no vector divides, the recomputing backward pass.
@pytest.mark.parametrize("rows, features, hidden", [(1, 256, 512), (300, 264, 600), (70, 131, 77),
                                                    (20000, 128, 520)])
def test_forward_and_backward(rows, features, hidden):
    g = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, dy = mk(rows, features), mk(rows, features)
    w, b = mk(features), mk(features)
    ws = [(mk(*s) * s[1] ** -0.5).bfloat16() for s in ((hidden, features), (hidden, features),
                                                       (features, hidden))]
    off = torch.tensor([5], device=DEV)

    def step():
        n, mean, rstd = cc.layer_norm_with_stats(x, w, b, out_dtype=torch.bfloat16)
        h, saved = cc.gated_feed_forward_with_saved(n, *ws)
        y = cc.dropout(h, 0.25, 3, off, residual=x)
        dh = cc.dropout(dy, 0.25, 3, off).bfloat16()
        dn, *dws = cc.gated_feed_forward_backward(dh, saved, n, *ws)
        return (y, *cc.layer_norm_backward(dn, x, mean, rstd, w), *dws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.copy_(mk(rows, features)), dy.copy_(mk(rows, features)), off.add_(1)
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(got, step()))
