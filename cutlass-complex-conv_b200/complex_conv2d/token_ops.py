"""Operators on rows of features: layer norm, a gated feed-forward block and
dropout from a counter-based generator.

They are what follows a ``ComplexConv2d`` in a token-wise block: the NHWC
planes of ``forward_planar`` are rows of channels, one per pixel, and

    out = dropout(gated_feed_forward(layer_norm(x), ...), p, seed, residual=x)

runs on those rows with the library's kernels.  The reference has none of
these.  Inputs are CUDA tensors ``[..., features]``; rows with a common stride
are read in place, other layouts are made contiguous first.  Every function is
asynchronous on the current stream and differentiable; the ``*_backward``
functions are the gradients themselves, for callers that keep their own tape.
"""

import collections
import weakref

import torch
from torch import nn

from ._extension import cutlass_complex_conv as _C
from ._tangents import refuse_tangents

__all__ = [
    "layer_norm", "layer_norm_with_stats", "layer_norm_backward",
    "gated_feed_forward", "gated_feed_forward_with_saved", "gated_feed_forward_backward",
    "dropout", "LayerNorm", "GatedFeedForward", "Dropout",
]

_U64 = (1 << 64) - 1


# ------------------------------------------------------------------ layer norm
def layer_norm_with_stats(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """``layer_norm`` without autograd: ``(y, mean, rstd)``, the statistics in
    float32 with one element per row."""
    return _C.layer_norm_forward(x, weight, bias, eps, out_dtype, True)


def layer_norm_backward(dy, x, mean, rstd, weight=None):
    """Gradients ``(dx, dweight, dbias)`` of ``layer_norm`` from the upstream
    gradient and the forward's statistics.  ``dweight`` and ``dbias`` have the
    weight's type (float32 without a weight); deterministic."""
    return _C.layer_norm_backward(dy, x, mean, rstd, weight, None, True, True, True)


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, mean, rstd = _C.layer_norm_forward(x, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        refuse_tangents("the gradient of layer_norm", dy)
        x, mean, rstd, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _C.layer_norm_backward(dy, x, mean, rstd, weight, ctx.bias_dtype, need[0],
                                            need[1], need[2])
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """Layer norm over the last dimension,
    ``(x - mean) / sqrt(var + eps) * weight + bias``.

    ``x``: float32, bfloat16 or float16; ``weight`` and ``bias``: float32 or
    x's type, or None.  The result has x's type; ``out_dtype`` asks for
    float32 from a 16-bit input, or for any of the three from float32 (so
    float32 planes can feed a 16-bit block without a copy).
    """
    refuse_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFunction.apply(x, weight, bias, eps, out_dtype)
    return _C.layer_norm_forward(x, weight, bias, eps, out_dtype, False)[0]


# ------------------------------------------------------------------ gated feed-forward
def gated_feed_forward_with_saved(x, w_gate, w_up, w_down, activation="silu"):
    """``gated_feed_forward`` without autograd: ``(y, saved)``, where ``saved``
    is the buffer ``gated_feed_forward_backward`` reads."""
    return _C.gated_ffn_forward(x, w_gate, w_up, w_down, activation, True)


def gated_feed_forward_backward(dy, saved, x, w_gate, w_up, w_down, activation="silu"):
    """Gradients ``(dx, dw_gate, dw_up, dw_down)`` of ``gated_feed_forward``;
    deterministic."""
    return _C.gated_ffn_backward(dy, saved, x, w_gate, w_up, w_down, activation, True, True, True,
                                 True)


class _GatedFeedForwardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        y, saved = _C.gated_ffn_forward(x, w_gate, w_up, w_down, activation, True)
        ctx.save_for_backward(saved, x, w_gate, w_up, w_down)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        refuse_tangents("the gradient of gated_feed_forward", dy)
        need = ctx.needs_input_grad
        return (*_C.gated_ffn_backward(dy, *ctx.saved_tensors, ctx.activation, need[0], need[1],
                                       need[2], need[3]), None)


def gated_feed_forward(x, w_gate, w_up, w_down, activation="silu"):
    """Gated feed-forward block
    ``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``.

    ``x [..., features]``, ``w_gate`` and ``w_up [hidden, features]``,
    ``w_down [features, hidden]``, all bfloat16 or all float16 (the tensor
    cores' operand types; sums are in float32, and the hidden values between
    the products are rounded to the type, so in float16 they must stay within
    65504 and lose bits below 6e-5, in the gradients too).  ``activation``: ``"silu"`` or ``"gelu"`` (the exact form with erf).
    """
    refuse_tangents("gated_feed_forward", x, w_gate, w_up, w_down)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
        return _GatedFeedForwardFunction.apply(x, w_gate, w_up, w_down, activation)
    return _C.gated_ffn_forward(x, w_gate, w_up, w_down, activation, False)[0]


# ------------------------------------------------------------------ dropout
def _dropout(x, p, seed, offset, residual):
    if isinstance(offset, torch.Tensor):
        return _C.dropout(x, p, seed & _U64, 0, offset, residual)
    return _C.dropout(x, p, seed & _U64, offset & _U64, None, residual)


def _dropout_backward(dy, p, seed, offset, x_dtype):
    if dy.dtype == x_dtype:  # the same call on the gradient
        return _dropout(dy, p, seed, offset, None)
    if isinstance(offset, torch.Tensor):
        return _C.dropout_backward(dy, p, seed & _U64, 0, offset, x_dtype)
    return _C.dropout_backward(dy, p, seed & _U64, offset & _U64, None, x_dtype)


class _DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        # A tensor offset may be changed before the backward pass runs (that
        # is what it is for): the mask of this pass needs its present value.
        ctx.offset = offset.clone() if isinstance(offset, torch.Tensor) else offset
        ctx.p, ctx.seed, ctx.x_dtype = p, seed, x.dtype
        return _dropout(x, p, seed, offset, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        refuse_tangents("the gradient of dropout", dy)
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _dropout_backward(dy, ctx.p, ctx.seed, ctx.offset, ctx.x_dtype)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """Drops elements of ``x`` with probability ``p`` and scales the rest by
    the inverse of the share kept; ``residual`` (x's type or float32) is added
    in the same pass and gives the result its type.

    The mask is a function of ``(seed, offset)`` and the element's index
    (Philox4x32-10) and is never stored: the same call on a gradient is the
    backward pass.  The probability is rounded to a multiple of 1/65536.
    ``seed``: an int; ``offset``: an int, or an int64 CUDA tensor of one
    element that is read when the kernel runs, so that a captured graph draws
    a new mask on each replay after its owner has changed it.  Use another
    offset for each call of a step.
    """
    refuse_tangents("dropout", x, residual)
    if torch.is_grad_enabled() and (
            x.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutFunction.apply(x, residual, p, seed, offset)
    return _dropout(x, p, seed, offset, residual)


# ------------------------------------------------------------------ modules
class LayerNorm(nn.Module):
    """``layer_norm`` with float32 (or ``dtype``) parameters ``weight`` and
    ``bias``."""

    def __init__(self, features, eps=1e-5, bias=True, out_dtype=None, device=None, dtype=None):
        super().__init__()
        self.features, self.eps, self.out_dtype = features, eps, out_dtype
        self.weight = nn.Parameter(torch.ones(features, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(features, device=device, dtype=dtype)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps, self.out_dtype)

    def extra_repr(self):
        return f"{self.features}, eps={self.eps}, bias={self.bias is not None}"


class GatedFeedForward(nn.Module):
    """``gated_feed_forward`` with its three weights as parameters (bfloat16
    unless ``dtype`` says float16), initialised U(+-1/sqrt(fan_in))."""

    def __init__(self, features, hidden, activation="silu", device=None, dtype=torch.bfloat16):
        super().__init__()
        if activation not in ("silu", "gelu"):
            raise ValueError(f"activation must be 'silu' or 'gelu', got {activation!r}")
        self.features, self.hidden, self.activation = features, hidden, activation
        kw = {"device": device, "dtype": dtype}
        self.w_gate = nn.Parameter(torch.empty(hidden, features, **kw))
        self.w_up = nn.Parameter(torch.empty(hidden, features, **kw))
        self.w_down = nn.Parameter(torch.empty(features, hidden, **kw))
        self.reset_parameters()

    def reset_parameters(self):
        for w in (self.w_gate, self.w_up, self.w_down):
            bound = w.shape[1] ** -0.5
            nn.init.uniform_(w, -bound, bound)

    def forward(self, x):
        return gated_feed_forward(x, self.w_gate, self.w_up, self.w_down, self.activation)

    def extra_repr(self):
        return f"{self.features}, {self.hidden}, activation={self.activation!r}"


_CALLS_KEPT = 4096
# Keys of masks drawn from torch's seed, away from keys that callers choose.
_DRAWN = 0x9E3779B97F4A7C15


class _Call:
    """A call of a Dropout module that a backward pass may have to repeat."""

    __slots__ = "number", "node", "repeated"

    def __init__(self, number):
        self.number, self.node, self.repeated = number, None, False

    def over(self):
        """Whether nothing can ask for it any more: its graph is gone or, for
        a call that recorded none (reentrant checkpointing), it was repeated."""
        return self.repeated if self.node is None else self.node() is None


class _Calls(collections.OrderedDict):
    """A module's last calls, by the generator's state each began at:
    {state: [_Call]}.  Copies and pickles of a module start without any."""

    def __reduce__(self):
        return _Calls, ()


def _generator_state(device):
    """State of torch's generator for ``device``, which it moves on by one
    step; None while the current stream is captured (its state is on the
    device then)."""
    if device.type != "cuda":
        return device.type, 0, int(torch.randint(1 << 62, (), device=device))
    if torch.cuda.is_current_stream_capturing():
        return None
    generator = torch.cuda.default_generators[device.index]
    state = device.index, generator.initial_seed(), generator.get_offset()
    generator.set_offset(state[2] + 4)  # torch counts in fours
    return state


class Dropout(nn.Module):
    """``dropout`` with a new mask at each call in training mode.  In
    evaluation mode ``x`` passes (with ``residual`` added, if given).

    Without ``seed`` the masks are a function of torch's generator for x's
    device, as ``torch.nn.Dropout``'s are: each call moves it on, so modules
    draw different masks, processes seeded differently do too, and a saved
    generator state resumes the sequence.  With ``seed`` call n draws mask
    ``(seed, n)``, whatever the generator's seed: give each module and each
    process its own.  The count is in ``state_dict``.

    A call that activation checkpointing repeats draws its mask again: it
    finds the generator in the state it had then.  Where it does not
    (``preserve_rng_state=False``) the repetition raises ``RuntimeError``.  In
    a captured graph the offset is drawn on the device, so that each replay
    has new masks.  ``offset`` in the call (an int, or a tensor as in
    ``dropout``) replaces all that, and nothing is counted."""

    def __init__(self, p=0.1, seed=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be between 0 and 1, got {p}")
        self.p, self.seed, self.calls = p, seed, 0
        self._begun = _Calls()

    def forward(self, x, residual=None, offset=None):
        if not self.training or self.p == 0.0:
            # (The sum of two types is float32: rounded to the residual's, as in training.)
            return x if residual is None else (residual + x).to(residual.dtype)
        seed = _DRAWN if self.seed is None else self.seed
        if offset is not None:
            return dropout(x, self.p, seed, offset, residual)
        state = _generator_state(x.device)
        repeated = torch._C._current_graph_task_id() != -1  # inside a backward pass
        if state is None:
            if repeated:
                self._refuse("a stream is being captured")
            offset = torch.randint(1 << 62, (1,), device=x.device)
            return dropout(x, self.p, seed, offset, residual)
        call = self._repeated(state) if repeated else self._new(state)
        offset = call.number
        if self.seed is None:
            seed, offset = state[1] ^ _DRAWN, state[2]
        y = dropout(x, self.p, seed, offset, residual)
        if not repeated and y.grad_fn is not None:
            call.node = weakref.ref(y.grad_fn)
        return y

    def _new(self, state):
        call = _Call(self.calls)
        self.calls += 1
        before = self._begun.pop(state, None)
        self._begun[state] = [call] if before is None else [c for c in before if not c.over()] + [call]
        if len(self._begun) > _CALLS_KEPT:
            self._begun.popitem(last=False)
        return call

    def _repeated(self, state):
        calls = self._begun.get(state, [])
        calls = [c for c in calls if c.node is None or not c.over()] or calls
        if not calls:
            self._refuse("the generator is in no state that a forward call began at")
        if len(calls) > 1 and self.seed is not None:
            self._refuse("several calls began at this state of the generator")
        calls[-1].repeated = True
        return calls[-1]

    def _refuse(self, why):
        raise RuntimeError(
            f"Dropout was called inside a backward pass and cannot tell which call's mask to "
            f"repeat ({why}): pass offset=, or checkpoint with preserve_rng_state=True")

    def get_extra_state(self):
        return torch.tensor(self.calls, device="cpu")

    def set_extra_state(self, state):
        self.calls = int(state)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs)
        key = prefix + "_extra_state"
        if key in missing_keys:  # saved before the count was kept
            missing_keys.remove(key)

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"
