"""Layer norm, forward and backward, against the 64-bit definition."""

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, HF = torch.bfloat16, torch.float32, torch.float16
EPS = 1e-5
TYPES = [(FP, FP, FP), (FP, FP, BF), (FP, FP, HF), (BF, BF, BF), (BF, FP, BF), (BF, FP, FP),
         (BF, BF, FP), (HF, HF, HF), (HF, FP, HF)]


def _terms(features):
    """Float32 roundings on the longest chain: a lane sums up to features/32
    elements, then a tree, then a handful of operations per element."""
    return features / 32 + 40


def _inputs(rows, features, types, seed=0, mean=0.3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    tx, tw, ty = types
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = (mk(rows, features) * 1.5 + mean).to(tx)
    return x, (mk(features) * 0.2 + 1).to(tw), (mk(features) * 0.1).to(tw), mk(rows, features).to(ty)


def _check_forward(x, w, b, out, **kw):
    y, mean, rstd = cc.layer_norm_with_stats(x, w, b, EPS, out)
    ry, rmean, rrstd = ref.norm(x, w, b, EPS)
    t = _terms(x.shape[-1])
    xa = x.double().abs()
    ref.assert_bounded(mean, rmean, xa.mean(-1), t, "mean")
    # rstd moves by half the relative error of the variance, whose terms are
    # squares of differences from a rounded mean.
    spread = ((xa + rmean.abs()[..., None]).square().mean(-1)) * rrstd ** 3
    ref.assert_bounded(rstd, rrstd, rrstd + spread, t, "rstd")
    wa = w.double().abs() if w is not None else 1.0
    mag = ((xa + rmean.abs()[..., None] + xa.mean(-1, keepdim=True)) * rrstd[..., None]
           + ((x.double() - rmean[..., None]) * spread[..., None]).abs()) * wa
    if b is not None:
        mag = mag + b.double().abs()
    ref.assert_bounded(y, ry, mag, t, "y")
    return mean, rstd


def _check_backward(dy, x, mean, rstd, w):
    got = cc.layer_norm_backward(dy, x, mean, rstd, w)
    want, mags = ref.norm_backward(dy, x, mean, rstd, w)
    terms = (_terms(x.shape[-1]), 300, 300)  # rows are summed in chains of at most 256
    for name, g, r, m, t in zip(("dx", "dweight", "dbias"), got, want, mags, terms):
        ref.assert_bounded(g, r, m, t, name)
    return got


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(d)[6:] for d in t))
@pytest.mark.parametrize("rows, features", [(5, 64), (33, 250), (7, 1001), (130, 512)])
def test_types(rows, features, types):
    x, w, b, dy = _inputs(rows, features, types)
    mean, rstd = _check_forward(x, w, b, types[2])
    _check_backward(dy, x, mean, rstd, w)


@pytest.mark.parametrize("features", [1, 2, 7, 8, 31, 33, 96, 128, 256, 264, 520, 1000, 1024, 1032,
                                      2048, 2056, 4096, 5000, 8192, 8200, 16384, 16392, 40000])
@pytest.mark.parametrize("types", [(BF, FP, BF), (FP, FP, FP)], ids=["bf16", "f32"])
def test_widths(features, types):
    x, w, b, dy = _inputs(19, features, types, seed=features)
    mean, rstd = _check_forward(x, w, b, types[2])
    _check_backward(dy, x, mean, rstd, w)


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 147, 149, 1183, 1185, 5000, 20011])
@pytest.mark.parametrize("features", [48, 384])
def test_row_counts(rows, features):
    x, w, b, dy = _inputs(rows, features, (BF, BF, BF), seed=rows)
    mean, rstd = _check_forward(x, w, b, BF)
    _check_backward(dy, x, mean, rstd, w)


def test_no_rows():
    x = torch.empty(0, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    y, mean, rstd = cc.layer_norm_with_stats(x, w)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = cc.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_without_weight_or_bias():
    x, w, b, dy = _inputs(21, 320, (FP, FP, FP))
    mean, rstd = _check_forward(x, None, None, FP)
    _check_backward(dy, x, mean, rstd, None)
    _check_forward(x, None, b, FP)
    _check_forward(x, w, None, FP)


@pytest.mark.parametrize("offset, step", [(0, 1), (1, 1), (3, 1), (8, 2)])
def test_strided_and_misaligned_rows(offset, step):
    big, w, b, bigdy = _inputs(40, 400, (BF, FP, BF))
    x = big[::step, offset:offset + 264]
    dy = bigdy[::step, offset:offset + 264]
    mean, rstd = _check_forward(x, w[:264], b[:264], BF)
    _check_backward(dy, x, mean, rstd, w[:264])
    # One of the two strided, and a view whose weight starts off alignment.
    _check_backward(dy.contiguous(), x, mean, rstd, w[1:265])
    _check_forward(x, w[1:265], b[3:267], BF)


def test_leading_dimensions_and_transposed_input():
    x, w, b, _ = _inputs(4 * 6 * 5, 72, (FP, FP, FP))
    x4 = x.view(4, 6, 5, 72)
    y = cc.layer_norm(x4, w, b)
    assert torch.equal(y.view(-1, 72), cc.layer_norm(x, w, b))
    t = x4.transpose(0, 2)
    assert torch.equal(cc.layer_norm(t, w, b), cc.layer_norm(t.contiguous(), w, b))
    c = x.t().contiguous().t()  # features not adjacent
    assert torch.equal(cc.layer_norm(c, w, b), cc.layer_norm(x, w, b))


def test_large_mean_keeps_the_variance():
    """The variance is summed from differences, so a mean of 1000 times the
    spread costs no more than the rounding of x itself."""
    x, w, b, _ = _inputs(9, 1024, (FP, FP, FP), mean=1000.0)
    _check_forward(x, w, b, FP)


def test_constant_rows_and_special_values():
    x = torch.full((3, 96), 2.5, device=DEV)
    y, mean, rstd = cc.layer_norm_with_stats(x, eps=EPS)
    assert not y.any() and torch.equal(mean, x[:, 0])
    torch.testing.assert_close(rstd, torch.full_like(rstd, EPS ** -0.5))
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    y = cc.layer_norm(x)
    assert not y[0].any() and y[1].isnan().all() and y[2].isnan().any()


def test_gradients_match_differences():
    """Directional derivatives of the 64-bit forward against the kernel's
    gradients (float32: 1e-4 covers their rounding, 300 terms of 2^-24 each
    with cancellation between projections)."""
    x, w, b, dy = _inputs(17, 264, (FP, FP, FP))
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    cc.layer_norm(x, w, b, EPS).backward(dy)
    g = torch.Generator(device=DEV).manual_seed(5)
    for i, t in enumerate((x, w, b)):
        v = torch.randn(t.shape, generator=g, device=DEV, dtype=torch.double)
        h = 1e-5
        f = lambda s: (ref.norm(*(u.detach().double() + (s * v if u is t else 0)
                                  for u in (x, w, b)), EPS)[0] * dy.double()).sum()
        d = (f(h) - f(-h)) / (2 * h)
        scale = (t.grad.double() * v).abs().sum()
        assert abs(d - (t.grad.double() * v).sum()) <= 1e-4 * scale


def test_autograd_of_parts():
    x, w, b, dy = _inputs(40, 128, (BF, FP, BF))
    y, mean, rstd = cc.layer_norm_with_stats(x, w, b, EPS)
    dx, dw, db = cc.layer_norm_backward(dy, x, mean, rstd, w)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        ts = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
        out = cc.layer_norm(*ts, EPS)
        assert torch.equal(out, y)
        out.backward(dy)
        for t, want, n in zip(ts, (dx, dw, db), need):
            assert torch.equal(t.grad, want) if n else t.grad is None


def test_same_result_every_time_and_on_another_stream():
    x, w, b, dy = _inputs(3000, 1000, (BF, FP, BF))
    y, mean, rstd = cc.layer_norm_with_stats(x, w, b, EPS)
    first = cc.layer_norm_backward(dy, x, mean, rstd, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y2, m2, r2 = cc.layer_norm_with_stats(x, w, b, EPS)
        second = cc.layer_norm_backward(dy, x, m2, r2, w)
    s.synchronize()
    assert torch.equal(y, y2)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_refusals():
    x, w, b, dy = _inputs(4, 16, (FP, FP, FP))
    with pytest.raises(ValueError, match="one element per feature"):
        cc.layer_norm(x, w[:8], b)
    with pytest.raises(TypeError, match="float32 or of the input's type"):
        cc.layer_norm(x.bfloat16(), w.half(), b.half())
    with pytest.raises(TypeError, match="one type"):
        cc.layer_norm(x.bfloat16(), w.bfloat16(), b)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        cc.layer_norm(x.double())
    with pytest.raises(TypeError, match="16-bit input"):
        cc.layer_norm(x.bfloat16(), out_dtype=HF)
    with pytest.raises(ValueError, match="eps"):
        cc.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="at least one feature"):
        cc.layer_norm(torch.empty(3, 0, device=DEV))
    with pytest.raises(ValueError, match="device"):
        cc.layer_norm(x, w.cpu())
    y, mean, rstd = cc.layer_norm_with_stats(x, w, b)
    with pytest.raises(ValueError, match="shape"):
        cc.layer_norm_backward(dy[:, :8], x, mean, rstd, w)
    with pytest.raises(ValueError, match="one element per row"):
        cc.layer_norm_backward(dy, x, mean[:2], rstd[:2], w)
