"""Which mask a call of the ``Dropout`` module draws: recomputed calls
(activation checkpointing), several modules, resumed runs, captured graphs.

The draws are host code, so most of this runs on the CPU with the tests'
oracle in place of the kernel; the same checks run on the GPU with it."""

import copy
import pickle

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import token_reference as ref
import complex_conv2d as cc
from complex_conv2d import token_ops

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def _oracle(x, p, seed, offset, residual=None):
    y, _ = ref.dropout(x, p, seed, int(offset), residual)
    return y.to(x.dtype if residual is None else residual.dtype)


@pytest.fixture(params=DEVICES)
def device(request, monkeypatch):
    if request.param == "cpu":
        monkeypatch.setattr(token_ops, "_dropout", _oracle)
    torch.manual_seed(20)
    return request.param


def _x(device, n=64, seed=0):
    return torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(device)


def _mask(d, x):
    """The mask of the next call."""
    return d(torch.ones_like(x)) != 0


def _gradient(f, x):
    x = x.detach().clone().requires_grad_()
    y = f(x)
    y.sum().backward()
    return x.grad, y.detach()


@pytest.mark.parametrize("seed", [None, 4])
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_gradients_use_the_forward_masks(device, reentrant, seed):
    """y = d(x)^2, so dy/dx = 2 y / x where the element was kept; each segment
    holds two modules, and several segments are open at once."""
    a, b = cc.Dropout(0.5, seed), cc.Dropout(0.3, seed if seed is None else seed + 1)
    seen = []

    def block(t):
        seen.append(1)
        return b(a(t).square()) + t

    x = _x(device)
    rng = torch.cuda.get_rng_state() if device != "cpu" else torch.get_rng_state()
    grad, y = _gradient(lambda t: checkpoint(block, checkpoint(block, t, use_reentrant=reentrant),
                                             use_reentrant=reentrant), x)
    assert len(seen) == 4  # both segments were recomputed
    if seed is not None:
        assert a.calls == b.calls == 2
        a, b = cc.Dropout(0.5, seed), cc.Dropout(0.3, seed + 1)
    elif device == "cpu":
        torch.set_rng_state(rng)
    else:
        torch.cuda.set_rng_state(rng)
    plain, y2 = _gradient(lambda t: block(block(t)), x)
    assert torch.equal(y, y2) and torch.equal(grad, plain)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_of_several_steps_in_any_order(device, reentrant):
    """Two steps open at once, the first differentiated first; the generator
    seeded again before each step (its states repeat)."""
    d = cc.Dropout(0.5, 4)
    x = _x(device)
    for _ in range(3):
        torch.manual_seed(1)
        first = d.calls
        t = x.clone().requires_grad_()
        y = [checkpoint(lambda u: d(u).square(), t, use_reentrant=reentrant) for _ in range(2)]
        for i in (0, 1):
            (grad,) = torch.autograd.grad(y[i].sum(), t) if not reentrant else (_take(y[i], t),)
            m = ref.dropout(torch.ones_like(x), 0.5, 4, first + i)[1]
            assert torch.equal(grad != 0, m)


def _take(y, t):
    t.grad = None
    y.sum().backward()
    return t.grad


@pytest.mark.parametrize("seed", [None, 4])
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_without_the_generator_state_is_refused(device, reentrant, seed):
    """Where checkpointing does not restore the generator there is no telling
    which call is repeated."""
    d = cc.Dropout(0.5, seed)
    x = _x(device).requires_grad_()
    y = checkpoint(lambda t: d(t).square(), x, use_reentrant=reentrant, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match="offset"):
        y.sum().backward()
    # With the offset given there is nothing to restore.
    grad, y = _gradient(lambda t: checkpoint(lambda u: d(u, offset=3).square(), t,
                                             use_reentrant=reentrant, preserve_rng_state=False), x)
    assert torch.equal(grad != 0, y != 0)


def test_a_call_whose_result_leaves_no_graph_is_repeated_too(device):
    """Its node is gone when the segment is recomputed."""
    d = cc.Dropout(0.5, 4)
    grad, y = _gradient(lambda t: checkpoint(lambda u: (d(u).detach() != 0) * u.square(), t,
                                             use_reentrant=False), _x(device))
    assert torch.equal(grad != 0, y != 0)


def test_recomputation_that_could_be_either_of_two_calls_is_refused(device):
    d = cc.Dropout(0.5, 4)
    x = _x(device).requires_grad_()
    y = []
    for _ in range(2):
        torch.manual_seed(1)
        y.append(checkpoint(lambda t: d(t).square(), x, use_reentrant=False))
    with pytest.raises(RuntimeError, match="offset"):
        y[0].sum().backward()


def test_modules_of_one_network_draw_their_own_masks(device):
    x = _x(device, 4096)
    a, b, c = cc.Dropout(0.5), cc.Dropout(0.5), copy.deepcopy(cc.Dropout(0.5))
    masks = [_mask(d, x) for _ in range(2) for d in (a, b, c)]
    for i in range(6):
        for j in range(i):
            # Independent masks agree in half of 4096 elements, 32 the standard deviation.
            agree = int((masks[i] == masks[j]).sum())
            assert abs(agree - 2048) < 6 * 32


def test_masks_without_a_seed_follow_torch(device):
    """The same state of torch's generator, the same masks; another seed of
    it (another rank's), others."""
    x = _x(device, 4096)
    torch.manual_seed(5)
    first = _mask(cc.Dropout(0.5), x)
    torch.manual_seed(6)
    other = _mask(cc.Dropout(0.5), x)
    torch.manual_seed(5)
    assert torch.equal(_mask(cc.Dropout(0.5), x), first)
    assert abs(int((first == other).sum()) - 2048) < 6 * 32


def test_a_seed_and_its_call_count_name_the_mask(device):
    """Whatever else draws from the generator, and however it is seeded."""
    x = _x(device, 512)
    a, b = cc.Dropout(0.5, 4), cc.Dropout(0.5, 9)
    for n in range(3):
        torch.manual_seed(1)
        torch.rand(3, device=device)
        for d in (a, b):
            assert torch.equal(_mask(d, x), ref.dropout(torch.ones_like(x), 0.5, d.seed, n)[1])
        a.eval(), a(x), a.train()
    assert a.calls == b.calls == 3


def test_a_resumed_run_continues_the_sequence(device):
    x = _x(device, 512)
    a = cc.Dropout(0.5, 4)
    _mask(a, x), _mask(a, x)
    state = a.state_dict()
    want = _mask(a, x)
    b = cc.Dropout(0.5, 4)
    assert not torch.equal(_mask(b, x), want)
    b.load_state_dict(state)
    assert torch.equal(_mask(b, x), want)
    c = pickle.loads(pickle.dumps(a))
    assert torch.equal(_mask(c, x), _mask(a, x))
    # A state from before the count was kept.
    assert cc.Dropout(0.5, 4).load_state_dict({}, strict=True) is not None
    net = torch.nn.Sequential(torch.nn.Linear(2, 2), cc.Dropout(0.5, 4))
    net.load_state_dict({k: v for k, v in net.state_dict().items() if "0." in k}, strict=True)


def test_count_is_kept_on_the_host_whatever_the_default_device():
    """A state made or loaded under another default device."""
    a, b = cc.Dropout(0.5, 4), cc.Dropout(0.5, 4)
    a.calls = 7
    with torch.device("meta"):
        state = a.state_dict()
        b.load_state_dict(state)
    assert b.calls == 7


@pytest.mark.parametrize("seed", [None, 4])
@pytest.mark.parametrize("inner", [False, True])
@pytest.mark.parametrize("outer", [False, True])
def test_nested_segments(device, outer, inner, seed):
    d = cc.Dropout(0.5, seed)
    x = _x(device)
    seen = []

    def step(t):
        seen.append(t)
        return d(t).square()

    grad, y = _gradient(lambda t: checkpoint(
        lambda u: checkpoint(step, step(u), use_reentrant=inner) + u, t, use_reentrant=outer), x)
    # y = x + (2 (2 x)^2)^2 where both masks kept it: dy/dx = 1 + 4 (y - x) / x.
    want = 1 + 4 * (y.double() - x.double()) / x.double()
    assert len(seen) > 3  # how often is the checkpointing's affair
    assert torch.equal(grad == 1, y == x)
    torch.testing.assert_close(grad.double(), want, rtol=1e-4, atol=1e-4)


def test_memory_of_calls_is_bounded(device):
    d = cc.Dropout(0.5, 4)
    x = _x(device, 1)
    with torch.no_grad():
        for _ in range(token_ops._CALLS_KEPT + 50):
            d(x)
    assert len(d._begun) == token_ops._CALLS_KEPT
    assert len(copy.deepcopy(d)._begun) == len(pickle.loads(pickle.dumps(d))._begun) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [None, 4])
def test_replays_of_a_captured_graph_draw_new_masks(seed):
    d = cc.Dropout(0.5, seed)
    x = torch.ones(4096, device="cuda:0", requires_grad=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        d(x).sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    x.grad = None
    with torch.cuda.graph(g):
        y = d(x)
        y.sum().backward()
    masks = []
    for _ in range(3):
        x.grad.zero_()
        g.replay()
        torch.cuda.synchronize()
        masks.append(y.detach() != 0)
        assert torch.equal(x.grad, y.detach())  # the gradient's mask is the forward's
    for i in range(3):
        for j in range(i):
            assert abs(int((masks[i] == masks[j]).sum()) - 2048) < 6 * 32


@pytest.mark.gpu
def test_offset_on_the_device():
    d = cc.Dropout(0.5, 4)
    x = torch.ones(512, device="cuda:0")
    off = torch.tensor([7], device="cuda:0")
    assert torch.equal(d(x, offset=off), cc.dropout(x, 0.5, 4, 7)) and d.calls == 0
