"""64-bit definitions of the token operators, and the bounds the tests use.

Everything runs in float64 from the operators' formulas, on the device of the
inputs; the generator is restated with Python integers and numpy.
"""

import math

import numpy as np
import torch

# Unit roundoff of each type: half the distance from 1 to the next number.
ROUNDOFF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
F32 = 2.0 ** -24
# Half the smallest step of float16 near zero (the others have float32's range).
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


# ------------------------------------------------------------------ layer norm
def norm(x, weight, bias, eps):
    """(y, mean, rstd)."""
    x = x.double()
    mean = x.mean(-1)
    rstd = ((x - mean[..., None]).square().mean(-1) + eps).rsqrt()
    y = (x - mean[..., None]) * rstd[..., None]
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, mean, rstd


def norm_backward(dy, x, mean, rstd, weight):
    """(dx, dweight, dbias) and, for the bounds, the sums of magnitudes each
    is made of."""
    rows = x.reshape(-1, x.shape[-1]).double()
    g = dy.reshape(rows.shape).double()
    mu, r = mean.reshape(-1, 1).double(), rstd.reshape(-1, 1).double()
    z = (rows - mu) * r
    t = g if weight is None else g * weight.double()
    dx = r * (t - t.mean(1, keepdim=True) - z * (t * z).mean(1, keepdim=True))
    # |z| as its rounding sees it: x and mean may cancel.
    za = (rows.abs() + mu.abs()) * r
    mag_x = r * (t.abs() + t.abs().mean(1, keepdim=True)
                 + za * (t * z).abs().mean(1, keepdim=True)
                 + z.abs() * (t.abs() * za).mean(1, keepdim=True))
    return ((dx.reshape(x.shape), (g * z).sum(0), g.sum(0)),
            (mag_x.reshape(x.shape), (g.abs() * za).sum(0), g.abs().sum(0)))


def assert_bounded(got, ref, magnitude, terms, what=""):
    """|got - ref| <= one rounding to got's type + `terms` float32 roundings
    of the magnitudes summed."""
    u = ROUNDOFF[got.dtype]
    limit = u * ref.abs() + (terms * F32) * magnitude * (1 + u) + TINY[got.dtype]
    bad = ~((got.double() - ref).abs() <= limit)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
        f"{((got.double() - ref).abs() / limit.clamp_min(1e-300)).max().item():.2f} x")


# ------------------------------------------------------------------ feed-forward
def _act(g, name):
    """act(g), act'(g), act''(g)."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), s * (1 - s) * (2 + g * (1 - 2 * s))
    c = 0.5 * (1 + torch.special.erf(g / math.sqrt(2)))
    phi = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g * c, c + g * phi, phi * (2 - g * g)


def _rss(*pairs):
    """Root of the sum of squared products of a @ b, over the pairs."""
    return sum(a.square() @ b.square() for a, b in pairs).sqrt()


def ffn(x, w_gate, w_up, w_down, activation):
    """y and the root sum of squares of the products each element sums."""
    x, wg, wu, wd = (t.double() for t in (x, w_gate, w_up, w_down))
    h = _act(x @ wg.t(), activation)[0] * (x @ wu.t())
    return h @ wd.t(), _rss((h, wd.t()))


def ffn_backward(dy, x, w_gate, w_up, w_down, activation):
    """(dx, dw_gate, dw_up, dw_down) and their roots of summed squares.  In
    the latter dg and du stand with the magnitudes their rounded factors give
    them: a relative error e of g moves act(g) by g act'(g) e and act'(g) by
    g act''(g) e."""
    x, wg, wu, wd, dy = (t.double() for t in (x, w_gate, w_up, w_down, dy))
    x, dy = x.reshape(-1, x.shape[-1]), dy.reshape(-1, dy.shape[-1])
    g, u = x @ wg.t(), x @ wu.t()
    a, slope, curve = _act(g, activation)
    dh = dy @ wd
    dg, du, h = dh * u * slope, dh * a, a * u
    mg, mu = (dh * u).abs() * (slope.abs() + (g * curve).abs()), dh.abs() * (
        a.abs() + (g * slope).abs())
    return ((dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h),
            (_rss((mg, wg), (mu, wu)), _rss((mg.t(), x)), _rss((mu.t(), x)), _rss((dy.t(), h))))


def assert_product(got, ref, rss, what=""):
    """A result of the block's products, `rss` the root of the summed squares
    of the products it adds up.  Besides its own rounding (u |ref| at most)
    an element carries the independent roundings of its terms' factors - at
    most three of them (the intermediate, its gate and its up value), each of
    relative rms u / sqrt(3): an error of rms u rss.  Per element 6 rms are
    allowed (the largest of 10^7 normal errors is 5.3 rms), over all of them
    a root mean square of 1.5 u sqrt(ref^2 + rss^2)."""
    assert torch.isfinite(got).all(), what
    u = ROUNDOFF[got.dtype]
    err = got.double() - ref
    limit = u * ref.abs() + 6 * u * rss + TINY[got.dtype]
    worst = (err.abs() / limit.clamp_min(1e-300)).max().item()
    assert worst <= 1.0, f"{what}: worst element {worst:.2f} x the bound"
    if got.numel() >= 64:
        rms = err.square().mean().sqrt().item()
        most = 1.5 * u * (ref.square() + rss.square()).mean().sqrt().item() + TINY[got.dtype]
        assert rms <= most, f"{what}: rms error {rms:.2e}, bound {most:.2e}"


# ------------------------------------------------------------------ dropout
def philox(counter, key, rounds=10):
    """Philox4x32 (Salmon, Moraes, Dror, Shaw, 2011) with Python integers."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def parts(seed, offset, first, count):
    """16-bit parts of elements first .. first + count - 1."""
    seed &= (1 << 64) - 1
    offset &= (1 << 64) - 1
    out = []
    for group in range(first // 8, (first + count + 7) // 8):
        words = philox((group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32),
                       (seed & 0xFFFFFFFF, seed >> 32))
        for w in words:
            out += [w & 0xFFFF, w >> 16]
    skip = first % 8
    return np.array(out[skip:skip + count], dtype=np.int64)


def threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def dropout(x, p, seed, offset, residual=None):
    t = threshold(p)
    keep = torch.from_numpy(parts(seed, offset, 0, x.numel()) >= t).to(x.device).reshape(x.shape)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    y = torch.where(keep, x.double() * scale, torch.zeros((), dtype=torch.double, device=x.device))
    return (y if residual is None else y + residual.double()), keep
