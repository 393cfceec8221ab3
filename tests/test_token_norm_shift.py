"""Layer norm's shifted vectors (dense rows of odd width): every element they
read lies in the tensor.  The values read beyond a row are masked, so no
result can show a read outside; the addresses are walked here on the CPU, with
the kernels' own arithmetic (csrc/ccv_norm_shift.h compiled for the host)."""

import ctypes
import os
import subprocess

import pytest
import torch

import token_reference as ref
import complex_conv2d as cc

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(cc.__file__))), "csrc")
SOURCE = """
#include "ccv_norm_shift.h"
using namespace ccv;
extern "C" {
int fits(int64_t features, int v) { return shift_fits(features, v); }
int shift(int64_t row, int features, int v) { return shift_of_row(row, features, v); }
int column(int i, int g, int lane, int v, int shift) { return shifted_column(i, g, lane, v, shift); }
int past(int64_t r, int64_t rows, int c, int features, int v) {
  return past_the_end(r, rows, c, features, v);
}
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    folder = tmp_path_factory.mktemp("shift")
    source, out = folder / "shift.cpp", folder / "shift.so"
    source.write_text(SOURCE)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC,
                           str(source), "-o", str(out)])
    lib = ctypes.CDLL(str(out))
    lib.fits.argtypes = [ctypes.c_int64, ctypes.c_int]
    lib.shift.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    lib.past.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    return lib


def _reads(lib, rows, features, v):
    """(row, first element, count, by element) of every fetch, as the kernels'
    fetch makes them; elements counted from the tensor's start."""
    need = -(-(features + v - 1) // 16)
    g = 1 << (need - 1).bit_length() if need <= 32 else -(-need // 32) * 32
    for r in range(rows):
        shift = lib.shift(r, features, v)
        for lane in range(g):
            for i in range(16 // v):
                c = lib.column(i, g, lane, v, shift)
                if lib.past(r, rows, c, features, v):
                    yield r, r * features + c, max(0, min(v, features - c)), True
                elif c < features:
                    yield r, r * features + c, v, False


def _outside(lib, rows, features, v):
    return [f for f in _reads(lib, rows, features, v)
            if f[2] and (f[1] < 0 or f[1] + f[2] > rows * features)]


WIDTHS = [1, 3, 5, 7, 9, 15, 17, 31, 33, 41, 505, 1001]


@pytest.mark.parametrize("v", [4, 8])
@pytest.mark.parametrize("features", WIDTHS)
def test_shifted_vectors_stay_in_the_tensor(lib, features, v):
    if not lib.fits(features, v):
        return  # such rows take single elements
    for rows in (1, 2, 3, 8, 9, 10, 17):
        assert _outside(lib, rows, features, v) == []
        seen = [[0] * features for _ in range(rows)]
        for r, first, count, by_element in _reads(lib, rows, features, v):
            assert by_element or first % v == 0, "a vector load off alignment"
            for e in range(max(first, r * features), min(first + count, (r + 1) * features)):
                seen[r][e - r * features] += 1
        assert all(n == 1 for row in seen for n in row)


def test_the_walk_sees_a_read_outside(lib):
    """Widths that the rule refuses would read past the tensor's end."""
    refused = [(f, v) for f in WIDTHS for v in (4, 8) if not lib.fits(f, v)]
    assert refused == [(1, 4), (1, 8), (3, 8), (5, 8)]
    for features, v in refused:
        assert any(_outside(lib, rows, features, v) for rows in range(2, 12))


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.bfloat16, torch.float32),
                                   (torch.float32, torch.float32, torch.float16),
                                   (torch.float32, torch.float32, torch.float32)],
                         ids=lambda t: "-".join(str(d)[6:] for d in t))
@pytest.mark.parametrize("features", [1, 3, 5, 7])
@pytest.mark.parametrize("rows", [2, 9, 20001])
def test_narrow_rows_in_front_of_foreign_memory(rows, features, types):
    """Rows followed at once by NaN that is not theirs."""
    tx, tw, ty = types
    gen = torch.Generator(device="cuda:0").manual_seed(features)
    n = rows * features

    def rows_of(dtype):
        t = torch.full((n + 64,), float("nan"), device="cuda:0", dtype=dtype)
        t[:n] = torch.randn(n, generator=gen, device="cuda:0").to(dtype)
        return t[:n].view(rows, features)

    x, dy = rows_of(tx), rows_of(ty)
    w = (torch.randn(features, generator=gen, device="cuda:0") * 0.2 + 1).to(tw)
    b = torch.randn(features, generator=gen, device="cuda:0").to(tw)
    y, mean, rstd = cc.layer_norm_with_stats(x, w, b, 0.1, ty)
    want, _, wrstd = ref.norm(x, w, b, 0.1)
    # A handful of float32 roundings (at most 7 terms a sum) of magnitudes
    # that rstd (at most 0.1^-1/2) scales; mean and x may cancel.
    mag = (x.double().abs().amax(1, keepdim=True) * 4 * wrstd[:, None]
           * (1 + x.double().square().amax(1, keepdim=True) * 4 * wrstd[:, None] ** 2)
           * w.double().abs() + b.double().abs())
    ref.assert_bounded(y, want, mag, 40, "y")
    got = cc.layer_norm_backward(dy, x, mean, rstd, w)
    want, mags = ref.norm_backward(dy, x, mean, rstd, w)
    for name, g, r, m, t in zip(("dx", "dweight", "dbias"), got, want, mags, (40, 300, 300)):
        ref.assert_bounded(g, r, m, t, name)
