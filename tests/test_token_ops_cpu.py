"""Refusals of the token operators that need no GPU: the C ABI's argument
checks come before any launch, and the Python entry points refuse CPU
tensors."""

import ctypes

import pytest
import torch

import ccv_abi
import complex_conv2d as cc

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
F32, BF16, F16 = 0, 1, 2


def _call(name, *args):
    """Calls a C entry point with typed scalars; returns (status, message)."""
    ccv_abi.load()
    f = getattr(ctypes.CDLL(ccv_abi.LIB), name)
    f.restype = ctypes.c_int
    typed = []
    for a in args:
        if a is None:
            typed.append(ctypes.c_void_p(None))
        elif isinstance(a, float):
            typed.append(ctypes.c_float(a))
        elif isinstance(a, int):
            typed.append(ctypes.c_int64(a))
        else:
            typed.append(a)
    return f(*typed), ccv_abi.last_error()


P = ctypes.c_void_p(0x1000)   # an aligned address; never dereferenced by the checks
ODD = ctypes.c_void_p(0x1001)


def _i(v):
    return ctypes.c_int(v)


def _norm(x=P, xt=F32, stride=8, w=P, b=P, wt=F32, eps=1e-5, y=P, yt=F32, rows=4, features=8):
    return _call("ccv_layer_norm_forward", x, _i(xt), stride, w, b, _i(wt), eps, y, _i(yt), None,
                 None, rows, features, None)


@pytest.mark.parametrize("kw, status, text", [
    (dict(rows=-1), INVALID, "rows"),
    (dict(features=0), INVALID, "features"),
    (dict(xt=7), INVALID, "element type"),
    (dict(xt=BF16, wt=F16, yt=BF16), INVALID, "weights"),
    (dict(xt=F32, wt=BF16), INVALID, "weights"),
    (dict(xt=BF16, yt=F16), INVALID, "16-bit input"),
    (dict(eps=-1.0), INVALID, "eps"),
    (dict(eps=float("nan")), INVALID, "eps"),
    (dict(x=None), INVALID, "null"),
    (dict(y=None), INVALID, "null"),
    (dict(x=ODD), INVALID, "aligned"),
    (dict(stride=-8), INVALID, "stride"),
    (dict(rows=1 << 40), UNSUPPORTED, "too large"),
])
def test_layer_norm_refusals(kw, status, text):
    rc, msg = _norm(**kw)
    assert rc == status and text in msg


def test_layer_norm_of_no_rows_launches_nothing():
    assert _norm(x=None, y=None, rows=0)[0] == 0


def _ffn(x=P, y=P, w=P, dtype=BF16, act=0, rows=4, features=8, hidden=16, saved=None,
         saved_bytes=0, ws=P, ws_bytes=1 << 20):
    size = lambda v: ctypes.c_size_t(v)
    return _call("ccv_gated_ffn_forward", x, 8, w, P, P, y, _i(dtype), _i(act), rows, features,
                 hidden, saved, size(saved_bytes), ws, size(ws_bytes), None)


@pytest.mark.parametrize("kw, status, text", [
    (dict(dtype=F32), INVALID, "bfloat16 or float16"),
    (dict(act=9), INVALID, "activation"),
    (dict(hidden=0), INVALID, "hidden"),
    (dict(features=-3), INVALID, "features"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(x=None), INVALID, "null"),
    (dict(w=None), INVALID, "null"),
    (dict(x=ODD), INVALID, "aligned"),
    (dict(saved=P, saved_bytes=8), WORKSPACE, "saved"),
    (dict(ws=None), WORKSPACE, "workspace"),
    (dict(ws_bytes=0), WORKSPACE, "workspace"),
    (dict(rows=1 << 33), UNSUPPORTED, "too large"),
])
def test_feed_forward_refusals(kw, status, text):
    rc, msg = _ffn(**kw)
    assert rc == status and text in msg


def test_feed_forward_of_no_rows_launches_nothing():
    assert _ffn(x=None, y=None, rows=0)[0] == 0


def _drop(x=P, xt=F32, r=None, y=P, yt=F32, count=8, p=0.5):
    u64 = ctypes.c_uint64
    return _call("ccv_dropout", x, _i(xt), r, y, _i(yt), count, ctypes.c_double(p), u64(1), u64(2),
                 None, None)


@pytest.mark.parametrize("kw, text", [
    (dict(p=-0.1), "p must"), (dict(p=1.5), "p must"), (dict(p=float("nan")), "p must"),
    (dict(count=-1), "count"), (dict(xt=5), "element type"), (dict(yt=BF16), "without a residual"),
    (dict(xt=BF16, yt=F16, r=P), "residual of its own"), (dict(x=None), "null"),
    (dict(y=ODD), "aligned"),
])
def test_dropout_refusals(kw, text):
    rc, msg = _drop(**kw)
    assert rc == INVALID and text in msg


def test_dropout_of_nothing_launches_nothing():
    assert _drop(x=None, y=None, count=0)[0] == 0


def test_python_entry_points_refuse_cpu_tensors():
    x = torch.zeros(2, 8)
    w = torch.zeros(16, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        cc.layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        cc.gated_feed_forward(x.bfloat16(), w, w, w.t())
    with pytest.raises(ValueError, match="CUDA"):
        cc.dropout(x, 0.5, 1)


def test_modules_refuse_bad_arguments_and_keep_their_parameters():
    with pytest.raises(ValueError, match="activation"):
        cc.GatedFeedForward(8, 16, activation="relu")
    with pytest.raises(ValueError, match="p must"):
        cc.Dropout(1.5)
    assert set(cc.LayerNorm(8).state_dict()) == {"weight", "bias"}
    assert set(cc.LayerNorm(8, bias=False).state_dict()) == {"weight"}
    ffn = cc.GatedFeedForward(8, 16)
    assert set(ffn.state_dict()) == {"w_gate", "w_up", "w_down"}
    assert ffn.w_down.shape == (8, 16) and ffn.w_gate.dtype == torch.bfloat16


def test_dropout_module_counts_its_calls_only_in_training():
    d = cc.Dropout(0.5, seed=3).eval()
    x = torch.ones(4)
    assert d(x) is x and d.calls == 0
    assert torch.equal(d(x, residual=x), 2 * x)
