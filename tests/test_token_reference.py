"""CPU checks of the token operators' oracle: the generator against published
vectors, the gradients against central differences."""

import pytest
import torch

import token_reference as ref


@pytest.mark.parametrize("counter, key, words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_known_answers(counter, key, words):
    assert tuple(ref.philox(counter, key)) == words


def _difference(f, tensors, which, direction, step=1e-5):
    plus = [t + step * direction if i == which else t for i, t in enumerate(tensors)]
    minus = [t - step * direction if i == which else t for i, t in enumerate(tensors)]
    return (f(*plus) - f(*minus)) / (2 * step)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_feed_forward_gradients_match_differences(activation):
    gen = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=gen, dtype=torch.double)
    ts = [mk(5, 6), mk(9, 6), mk(9, 6), mk(6, 9)]
    dy = mk(5, 6)
    grads, _ = ref.ffn_backward(dy, *ts, activation)
    for i, g in enumerate(grads):
        v = mk(*ts[i].shape)
        d = _difference(lambda *a: (ref.ffn(*a, activation)[0] * dy).sum(), ts, i, v)
        assert abs(d - (g * v).sum()) <= 1e-6 * (1 + abs(d))


def test_layer_norm_gradients_match_differences():
    gen = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=gen, dtype=torch.double)
    ts = [mk(4, 7), mk(7), mk(7)]
    dy = mk(4, 7)
    _, mean, rstd = ref.norm(*ts, 1e-5)
    grads, _ = ref.norm_backward(dy, ts[0], mean, rstd, ts[1])
    for i, g in enumerate(grads):
        v = mk(*ts[i].shape)
        d = _difference(lambda *a: (ref.norm(*a, 1e-5)[0] * dy).sum(), ts, i, v)
        assert abs(d - (g * v).sum()) <= 1e-6 * (1 + abs(d))
