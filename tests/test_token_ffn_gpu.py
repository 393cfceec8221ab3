"""Gated feed-forward block, forward and backward, against the 64-bit
definition."""

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def _inputs(rows, features, hidden, dtype=BF, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return (mk(rows, features).to(dtype), (mk(hidden, features) * features ** -0.5).to(dtype),
            (mk(hidden, features) * features ** -0.5).to(dtype),
            (mk(features, hidden) * hidden ** -0.5).to(dtype), mk(rows, features).to(dtype))


def _check(x, wg, wu, wd, dy, activation, backward=True):
    y = cc.gated_feed_forward(x, wg, wu, wd, activation)
    ref.assert_product(y, *ref.ffn(x, wg, wu, wd, activation), "y")
    if not backward:
        return
    y2, saved = cc.gated_feed_forward_with_saved(x, wg, wu, wd, activation)
    ref.assert_product(y2, *ref.ffn(x, wg, wu, wd, activation), "y with saved")
    got = cc.gated_feed_forward_backward(dy, saved, x, wg, wu, wd, activation)
    want, rss = ref.ffn_backward(dy, x, wg, wu, wd, activation)
    for name, a, b, r in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want, rss):
        ref.assert_product(a, b, r, name)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows, features, hidden", [(64, 128, 256), (200, 264, 520)])
def test_types_and_activations(rows, features, hidden, activation, dtype):
    _check(*_inputs(rows, features, hidden, dtype), activation)


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 9, 16, 17, 24, 31, 32, 33, 64, 65, 127, 128, 129, 255,
                                  256, 257, 385, 600])
def test_row_counts(rows):
    _check(*_inputs(rows, 192, 328, seed=rows), "silu")


@pytest.mark.parametrize("features, hidden", [(8, 8), (64, 64), (72, 136), (128, 1000), (256, 1024),
                                              (520, 264), (1032, 2056), (2048, 512)])
@pytest.mark.parametrize("rows", [3, 300])
def test_widths(rows, features, hidden):
    _check(*_inputs(rows, features, hidden, seed=features), "gelu")


@pytest.mark.parametrize("features, hidden", [(1, 1), (7, 9), (65, 131), (129, 264), (136, 515),
                                              (1001, 333)])
@pytest.mark.parametrize("rows", [1, 40, 261])
def test_widths_that_no_vector_divides(rows, features, hidden):
    _check(*_inputs(rows, features, hidden, seed=hidden), "silu")


@pytest.mark.parametrize("rows, features, hidden", [(6000, 256, 512), (1, 1024, 4096),
                                                    (4, 2048, 5504), (2100, 512, 2048),
                                                    (25000, 128, 1000)])
def test_larger(rows, features, hidden):
    _check(*_inputs(rows, features, hidden, seed=rows), "silu")


@pytest.fixture
def switches(monkeypatch):
    """Sets the library's CCV_* switches for one test."""
    from complex_conv2d import _C

    def set_to(**kw):
        for k, v in kw.items():
            monkeypatch.setenv(k, str(v))
        _C.reload_config()

    yield set_to
    monkeypatch.undo()
    _C.reload_config()


@pytest.mark.parametrize("env", [
    dict(CCV_FFN_BN=128), dict(CCV_FFN_BN=256), dict(CCV_FFN_BN=256, CCV_FFN_SPLITS=3),
    dict(CCV_FFN_BN=128, CCV_FFN_SPLITS=5), dict(CCV_FFN_SPLITS=1)],
    ids=lambda e: "-".join(f"{k[8:]}{v}" for k, v in e.items()))
@pytest.mark.parametrize("rows, features, hidden", [(33, 64, 136), (300, 200, 1000), (1000, 264, 600),
                                                    (5000, 328, 1032), (257, 131, 77)])
def test_every_kernel(rows, features, hidden, env, switches):
    """Each tile width and the split of the last wave, on shapes they would
    not all be chosen for."""
    switches(**env)
    _check(*_inputs(rows, features, hidden, seed=hidden), "gelu")


def test_no_rows():
    x, wg, wu, wd, dy = _inputs(0, 64, 96)
    y, saved = cc.gated_feed_forward_with_saved(x, wg, wu, wd)
    assert y.shape == (0, 64)
    dx, *dws = cc.gated_feed_forward_backward(dy, saved, x, wg, wu, wd)
    assert dx.shape == (0, 64)
    assert all(w.shape == d.shape and not d.any() for w, d in zip((wg, wu, wd), dws))


@pytest.mark.parametrize("rows", [5, 150])
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
def test_strided_and_misaligned_rows(offset, rows):
    big, wg, wu, wd, bigdy = _inputs(rows, 400, 200)
    x, dy = big[:, offset:offset + 136], bigdy[:, offset:offset + 136]
    wg, wu, wd = wg[:, :136], wu[:, 8:144], wd[:136].clone()
    _check(x, wg, wu, wd, dy, "silu")
    # Weights whose storage starts off alignment.
    flat = torch.empty(200 * 136 + 1, device=DEV, dtype=BF)
    flat[1:] = wg.reshape(-1)
    _check(x, flat[1:].view(200, 136), wu, wd, dy, "silu")


def test_leading_dimensions():
    x, wg, wu, wd, dy = _inputs(60, 72, 96)
    y = cc.gated_feed_forward(x.view(3, 4, 5, 72), wg, wu, wd)
    assert torch.equal(y.view(60, 72), cc.gated_feed_forward(x, wg, wu, wd))


@pytest.mark.parametrize("rows", [1, 12, 200])
def test_special_values_stay_in_their_row(rows):
    x, wg, wu, wd, _ = _inputs(rows + 2, 64, 96)
    clean = cc.gated_feed_forward(x, wg, wu, wd)
    x[1] = float("nan")
    y = cc.gated_feed_forward(x, wg, wu, wd)
    assert y[1].isnan().all()
    keep = torch.arange(rows + 2, device=DEV) != 1
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_saturated_gates(activation):
    """Gates of +-200: the activation is the identity or zero, never NaN."""
    x, wg, wu, wd, dy = _inputs(40, 64, 96)
    _check(x, (wg.float() * 200).to(BF), wu, wd, dy, activation)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gradients_match_differences(activation):
    """Directional derivatives of the 64-bit forward against the kernel's
    gradients.  Elements with independent errors of rms 1.5 u |grad| / sqrt(N)
    move the projection on a unit-variance direction by 1.5 u |grad|; four
    times that is allowed."""
    x, wg, wu, wd, dy = _inputs(100, 128, 192)
    ts = [t.requires_grad_() for t in (x, wg, wu, wd)]
    cc.gated_feed_forward(*ts, activation).backward(dy)
    g = torch.Generator(device=DEV).manual_seed(5)
    for t in ts:
        v = torch.randn(t.shape, generator=g, device=DEV, dtype=torch.double)
        h = 1e-5
        f = lambda s: (ref.ffn(*(u.detach().double() + (s * v if u is t else 0) for u in ts),
                               activation)[0] * dy.double()).sum()
        d = (f(h) - f(-h)) / (2 * h)
        grad = t.grad.double()
        assert abs(d - (grad * v).sum()) <= 6 * ref.ROUNDOFF[BF] * grad.norm()


def test_autograd_of_parts():
    x, wg, wu, wd, dy = _inputs(70, 128, 256)
    y, saved = cc.gated_feed_forward_with_saved(x, wg, wu, wd)
    full = cc.gated_feed_forward_backward(dy, saved, x, wg, wu, wd)
    for need in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 1, 1)):
        ts = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, wg, wu, wd), need)]
        cc.gated_feed_forward(*ts).backward(dy)
        for t, want, n in zip(ts, full, need):
            assert torch.equal(t.grad, want) if n else t.grad is None


@pytest.mark.parametrize("rows, features, hidden", [(7, 256, 512), (3000, 256, 512),
                                                    (20000, 128, 520), (5000, 520, 1032)])
def test_same_result_every_time_and_on_another_stream(rows, features, hidden):
    x, wg, wu, wd, dy = _inputs(rows, features, hidden)

    def once():
        y, saved = cc.gated_feed_forward_with_saved(x, wg, wu, wd)
        return (y, *cc.gated_feed_forward_backward(dy, saved, x, wg, wu, wd))

    first = once()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = once()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_first_cuda_work_of_a_host_thread():
    """A thread that has made no CUDA call yet (its memory comes from the
    caching allocator) can run the block."""
    import threading
    args = _inputs(100, 128, 256)[:4]
    want = cc.gated_feed_forward(*args)
    torch.cuda.synchronize()
    got = []
    t = threading.Thread(target=lambda: got.append(cc.gated_feed_forward(*args)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_refusals():
    x, wg, wu, wd, dy = _inputs(4, 16, 24)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        cc.gated_feed_forward(x.float(), wg.float(), wu.float(), wd.float())
    with pytest.raises(TypeError, match="input's type"):
        cc.gated_feed_forward(x, wg.half(), wu, wd)
    with pytest.raises(ValueError, match="w_gate"):
        cc.gated_feed_forward(x, wg.t(), wu, wd)
    with pytest.raises(ValueError, match="w_up"):
        cc.gated_feed_forward(x, wg, wu[:8], wd)
    with pytest.raises(ValueError, match="w_down"):
        cc.gated_feed_forward(x, wg, wu, wd.t())
    with pytest.raises(ValueError, match="activation"):
        cc.gated_feed_forward(x, wg, wu, wd, "relu")
    with pytest.raises(ValueError, match="device"):
        cc.gated_feed_forward(x, wg.cpu(), wu, wd)
    y, saved = cc.gated_feed_forward_with_saved(x, wg, wu, wd)
    with pytest.raises(ValueError, match="saved"):
        cc.gated_feed_forward_backward(dy[:2], saved, x[:2], wg, wu, wd)
    with pytest.raises(ValueError, match="shape"):
        cc.gated_feed_forward_backward(dy[:2], saved, x, wg, wu, wd)
