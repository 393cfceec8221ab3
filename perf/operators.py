"""Cases and plain forms of the token operators: layer norm, the gated
feed-forward block and counter-based dropout.

They are the token-wise half of a block that follows a complex convolution:
``forward_planar`` hands out NHWC planes, one row of features per pixel, and
``out = residual + dropout(feed_forward(layer_norm(x)))`` runs on those rows.

``run`` computes a case either with elementary torch operations in 32 bits
(``own`` false) or with the package's operators (``own`` true); ``exact``
restates each definition in 64 bits.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DEVICE = "cuda"
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_EPS = 1e-5

# The most work a drawn case may have, per operator (that of the largest listed case).
_MAX_NORM = 200704 * 256
_MAX_FFN_FORWARD = 8192 * 2048 * 8192
_MAX_FFN_TRAIN = 8192 * 2048 * 8192
_MAX_DROPOUT = 200704 * 256


def _package():
    path = os.path.join(_ROOT, "cutlass-complex-conv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import complex_conv2d
    return complex_conv2d


def listed():
    return [
        # Layer norm over a batch of 64 feature maps of 56 x 56 pixels, real and imaginary parts of
        # 128 channels side by side: fp32 planes in, bf16 rows out for the products that follow.
        {"name": "norm_forward_maps", "op": "norm", "direction": "forward", "rows": 200704,
         "features": 256, "dtype": "float32", "out": "bfloat16", "weight": "float32"},
        # Its backward pass in training: bf16 upstream gradient, fp32 input gradient.
        {"name": "norm_backward_maps", "op": "norm", "direction": "backward", "rows": 200704,
         "features": 256, "dtype": "float32", "out": "bfloat16", "weight": "float32"},
        # One 7 x 7 map of 512 channels in bf16: a call where latency counts.
        {"name": "norm_forward_small", "op": "norm", "direction": "forward", "rows": 49,
         "features": 512, "dtype": "bfloat16", "out": "bfloat16", "weight": "bfloat16"},
        # A ragged batch of rows whose width is no multiple of a vector load.
        {"name": "norm_backward_odd", "op": "norm", "direction": "backward", "rows": 12545,
         "features": 1001, "dtype": "bfloat16", "out": "bfloat16", "weight": "float32"},
        # One token of a served model: the weights are read once for a single row.
        {"name": "ffn_forward_token", "op": "ffn", "direction": "forward", "rows": 1,
         "features": 1024, "hidden": 4096, "dtype": "bfloat16", "activation": "silu"},
        # One 28 x 28 map and one extra token, a hidden width that is no multiple of a tile.
        {"name": "ffn_forward_ragged", "op": "ffn", "direction": "forward", "rows": 785,
         "features": 512, "hidden": 1368, "dtype": "bfloat16", "activation": "gelu"},
        # A long prompt or a large batch of maps through a wide block.
        {"name": "ffn_forward_large", "op": "ffn", "direction": "forward", "rows": 8192,
         "features": 2048, "hidden": 8192, "dtype": "bfloat16", "activation": "silu"},
        # Training step (forward and backward) on a batch of 8 maps of 56 x 56 pixels, in fp16.
        {"name": "ffn_train_maps", "op": "ffn", "direction": "train", "rows": 25088,
         "features": 256, "hidden": 1024, "dtype": "float16", "activation": "gelu"},
        # Training step of the wide block.
        {"name": "ffn_train_large", "op": "ffn", "direction": "train", "rows": 8192,
         "features": 2048, "hidden": 8192, "dtype": "bfloat16", "activation": "silu"},
        # Dropout of the block's bf16 branch added to the fp32 residual planes.
        {"name": "dropout_residual_maps", "op": "dropout", "count": 200704 * 256,
         "dtype": "bfloat16", "residual": "float32", "p": 0.1, "seed": 1234, "offset": 7},
        # The same mask applied to a bf16 gradient, an odd number of elements.
        {"name": "dropout_gradient_odd", "op": "dropout", "count": 25088 * 1001 + 3,
         "dtype": "bfloat16", "residual": "", "p": 0.1, "seed": 99, "offset": (1 << 33) + 5},
        # A few rows: a call where latency counts.
        {"name": "dropout_small", "op": "dropout", "count": 49 * 512,
         "dtype": "float32", "residual": "", "p": 0.25, "seed": (1 << 40) + 3, "offset": 0},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "ffn", "ffn", "dropout"])
    if op == "norm":
        features = _log_int(rng, 32, 8192)
        if rng.random() < 0.6:
            features = max(8, features // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(200704, _MAX_NORM // features)))
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        out = rng.choice(["bfloat16", "float32"]) if dtype == "float32" else dtype
        weight = rng.choice(["float32", dtype])
        return {"op": "norm", "direction": rng.choice(["forward", "backward"]), "rows": rows,
                "features": features, "dtype": dtype, "out": out, "weight": weight}
    if op == "ffn":
        direction = rng.choice(["forward", "forward", "train"])
        features = _log_int(rng, 64, 2048)
        hidden = _log_int(rng, features, min(8192, 4 * features))
        if rng.random() < 0.8:
            features, hidden = features // 8 * 8, hidden // 8 * 8
        most = _MAX_FFN_FORWARD if direction == "forward" else _MAX_FFN_TRAIN
        rows = _log_int(rng, 1 if direction == "forward" else 16,
                        max(16, min(25088, most // (features * hidden))))
        return {"op": "ffn", "direction": direction, "rows": rows, "features": features,
                "hidden": hidden, "dtype": rng.choice(["bfloat16", "float16"]),
                "activation": rng.choice(["silu", "gelu"])}
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    return {"op": "dropout", "count": _log_int(rng, 1000, _MAX_DROPOUT), "dtype": dtype,
            "residual": rng.choice(["", "float32", dtype]), "p": round(rng.uniform(0.0, 0.6), 3),
            "seed": rng.randrange(1 << 48), "offset": rng.randrange(1 << 36)}


def _inputs(case, seed):
    """The case's tensors, the same for the same seed."""
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)

    def normal(shape, dtype, std=1.0, mean=0.0):
        t = torch.randn(shape, generator=gen, device=_DEVICE)
        return t.mul_(std).add_(mean).to(_DTYPES[dtype])

    def uniform(shape, dtype, bound):
        t = torch.rand(shape, generator=gen, device=_DEVICE)
        return t.mul_(2 * bound).sub_(bound).to(_DTYPES[dtype])

    if case["op"] == "norm":
        rows, features = case["rows"], case["features"]
        t = {"x": normal((rows, features), case["dtype"], 1.5, 0.3),
             "weight": normal((features,), case["weight"], 0.2, 1.0),
             "bias": normal((features,), case["weight"], 0.1)}
        if case["direction"] == "backward":
            t["dy"] = normal((rows, features), case["out"])
            x = t["x"].float()
            t["mean"] = x.mean(dim=1)
            t["rstd"] = ((x - t["mean"][:, None]).square().mean(dim=1) + _EPS).rsqrt()
        return t
    if case["op"] == "ffn":
        rows, features, hidden = case["rows"], case["features"], case["hidden"]
        t = {"x": normal((rows, features), case["dtype"]),
             "w_gate": uniform((hidden, features), case["dtype"], features ** -0.5 * 1.7),
             "w_up": uniform((hidden, features), case["dtype"], features ** -0.5 * 1.7),
             "w_down": uniform((features, hidden), case["dtype"], hidden ** -0.5 * 1.7)}
        if case["direction"] == "train":
            t["dy"] = normal((rows, features), case["dtype"])
        return t
    t = {"x": normal((case["count"],), case["dtype"])}
    if case["residual"]:
        t["residual"] = normal((case["count"],), case["residual"])
    return t


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    if own:
        state["package"] = _package()
    return state


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _run_norm(state, case)
    if case["op"] == "ffn":
        return _run_ffn(state, case)
    return _run_dropout(state, case)


# ------------------------------------------------------------------ layer norm
def _run_norm(s, case):
    out = _DTYPES[case["out"]]
    if own:
        pkg = s["package"]
        if case["direction"] == "forward":
            return pkg.layer_norm_with_stats(s["x"], s["weight"], s["bias"], _EPS, out)
        return pkg.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    x, w = s["x"].float(), s["weight"].float()
    if case["direction"] == "forward":
        mean = x.mean(dim=1)
        centred = x - mean[:, None]
        rstd = (centred.square().mean(dim=1) + _EPS).rsqrt()
        y = centred * rstd[:, None] * w + s["bias"].float()
        return y.to(out), mean, rstd
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    t = dy * w
    dx = rstd * (t - t.mean(dim=1, keepdim=True)
                 - xhat * (t * xhat).mean(dim=1, keepdim=True))
    weight = s["weight"].dtype
    return dx.to(s["x"].dtype), (dy * xhat).sum(dim=0).to(weight), dy.sum(dim=0).to(weight)


def _exact_norm(t, case):
    x, w = t["x"].double(), t["weight"].double()
    n = x.shape[1]
    if case["direction"] == "forward":
        mean = x.sum(1) / n
        var = ((x - mean.view(-1, 1)) ** 2).sum(1) / n
        rstd = 1.0 / torch.sqrt(var + _EPS)
        return torch.addcmul(t["bias"].double(), (x - mean.view(-1, 1)) * rstd.view(-1, 1), w), \
            mean, rstd
    mean, rstd = t["mean"].double().view(-1, 1), t["rstd"].double().view(-1, 1)
    dy = t["dy"].double()
    z = (x - mean) * rstd
    dz = dy * w
    along = (dz * z).sum(1, keepdim=True) / n
    dx = (dz - dz.sum(1, keepdim=True) / n - z * along) * rstd
    return dx, (z * dy).sum(0), dy.sum(0)


# ------------------------------------------------------------------ gated feed-forward
def _run_ffn(s, case):
    act = case["activation"]
    if own:
        pkg = s["package"]
        weights = (s["w_gate"], s["w_up"], s["w_down"])
        if case["direction"] == "forward":
            with torch.no_grad():
                return pkg.gated_feed_forward(s["x"], *weights, activation=act)
        y, saved = pkg.gated_feed_forward_with_saved(s["x"], *weights, activation=act)
        return (y, *pkg.gated_feed_forward_backward(s["dy"], saved, s["x"], *weights,
                                                    activation=act))
    x = s["x"].float()
    w_gate, w_up, w_down = s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
    gate, up = x @ w_gate.t(), x @ w_up.t()
    if act == "silu":
        slope = 1.0 / (1.0 + torch.exp(-gate))          # sigmoid
        value = gate * slope
    else:
        slope = 0.5 * (1.0 + torch.erf(gate * 0.7071067811865476))   # normal distribution
        value = gate * slope
    hidden = value * up
    y = hidden @ w_down.t()
    dtype = s["x"].dtype
    if case["direction"] == "forward":
        return y.to(dtype)
    if act == "silu":
        slope = slope * (1.0 + gate * (1.0 - slope))
    else:
        slope = slope + gate * 0.3989422804014327 * torch.exp(-0.5 * gate * gate)
    dy = s["dy"].float()
    d_hidden = dy @ w_down
    d_gate, d_up = d_hidden * up * slope, d_hidden * value
    dx = d_gate @ w_gate + d_up @ w_up
    return (y.to(dtype), dx.to(dtype), (d_gate.t() @ x).to(dtype), (d_up.t() @ x).to(dtype),
            (dy.t() @ hidden).to(dtype))


def _exact_ffn(t, case):
    x, wg, wu, wd = (t[k].double() for k in ("x", "w_gate", "w_up", "w_down"))
    a, b = torch.mm(x, wg.T), torch.mm(x, wu.T)
    if case["activation"] == "silu":
        s = torch.sigmoid(a)
        d = s + a * s * (1 - s)
    else:
        s = torch.special.ndtr(a)
        d = s + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    f = a * s
    h = f * b
    y = torch.mm(h, wd.T)
    if case["direction"] == "forward":
        return y
    dy = t["dy"].double()
    e = torch.mm(dy, wd)
    da, db = e * b * d, e * f
    return y, torch.mm(da, wg) + torch.mm(db, wu), torch.mm(da.T, x), torch.mm(db.T, x), \
        torch.mm(dy.T, h)


# ------------------------------------------------------------------ dropout
# Element i takes 16 bits of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): key = the 64-bit
# seed, counter = (i // 8 in the low 64 bits, offset in the high 64); its eight 16-bit parts, low
# half of each word first, belong to elements 8k .. 8k + 7.  An element is dropped when its part is
# below round(p * 65536); the others are scaled by the inverse of the share that is kept.
_M0, _M1 = 0xD2511F53, 0xCD9E8D57
_W0, _W1 = 0x9E3779B9, 0xBB67AE85
_LOW = 0xFFFFFFFF


def _threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def _run_dropout(s, case):
    x, residual = s["x"], s.get("residual")
    if own:
        return s["package"].dropout(x, case["p"], case["seed"], case["offset"], residual=residual)
    limit = _threshold(case["p"])
    n = x.numel()
    c0 = torch.arange((n + 7) // 8, device=x.device, dtype=torch.int64)
    c1 = c0 >> 32
    c0 = c0 & _LOW
    c2 = torch.full_like(c0, case["offset"] & _LOW)
    c3 = torch.full_like(c0, (case["offset"] >> 32) & _LOW)
    k0, k1 = case["seed"] & _LOW, (case["seed"] >> 32) & _LOW
    for _ in range(10):
        p0, p1 = c0 * _M0, c2 * _M1
        c0, c1, c2, c3 = (((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW,
                          ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW)
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    words = torch.stack((c0, c1, c2, c3), dim=1)
    parts = torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:n]
    y = torch.where(parts >= limit, x.float() * (65536.0 / (65536 - limit)),
                    torch.zeros((), device=x.device))
    if residual is not None:
        return (y + residual.float()).to(residual.dtype)
    return y.to(x.dtype)


def _exact_dropout(t, case):
    n = case["count"]
    u64, low, half = np.uint64, np.uint64(_LOW), np.uint64(32)
    counter = np.arange(-(-n // 8), dtype=np.uint64)
    ctr = [counter & low, counter >> half, u64(case["offset"] & _LOW), u64(case["offset"] >> 32)]
    ctr = [np.broadcast_to(c, counter.shape) for c in ctr]
    key = [case["seed"] & _LOW, case["seed"] >> 32]
    for r in range(10):
        a, b = ctr[0] * u64(_M0), ctr[2] * u64(_M1)
        ka = u64((key[0] + r * _W0) & _LOW)
        kb = u64((key[1] + r * _W1) & _LOW)
        ctr = [(b >> half) ^ ctr[1] ^ ka, b & low, (a >> half) ^ ctr[3] ^ kb, a & low]
    bits = np.stack(ctr, axis=1).astype("<u4").view("<u2").reshape(-1)[:n]
    limit = _threshold(case["p"])
    keep = torch.from_numpy(bits.astype(np.int32)).to(t["x"].device) >= limit
    y = t["x"].double() * 65536.0 / (65536 - limit)
    y.masked_fill_(~keep, 0.0)
    if "residual" in t:
        y += t["residual"].double()
    return y


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(t, case)
    if case["op"] == "ffn":
        return _exact_ffn(t, case)
    return _exact_dropout(t, case)


def work(case):
    if case["op"] == "norm":
        n, d = case["rows"] * case["features"], case["features"]
        x, o, w = _BYTES[case["dtype"]], _BYTES[case["out"]], _BYTES[case["weight"]]
        if case["direction"] == "forward":
            return {"bytes": n * (x + o) + 2 * d * w + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": n * (2 * x + o) + 3 * d * w + 8 * case["rows"], "flops": 14 * n}
    if case["op"] == "ffn":
        m, d, f, e = case["rows"], case["features"], case["hidden"], _BYTES[case["dtype"]]
        if case["direction"] == "forward":
            return {"bytes": e * (2 * m * d + 3 * d * f), "flops": 6 * m * d * f}
        return {"bytes": e * (4 * m * d + 6 * d * f), "flops": 18 * m * d * f}
    n, e = case["count"], _BYTES[case["dtype"]]
    if case["residual"]:
        return {"bytes": n * (e + 2 * _BYTES[case["residual"]]), "flops": 2 * n}
    return {"bytes": 2 * n * e, "flops": n}
