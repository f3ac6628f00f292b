"""CPU: frequencies of rotary positions and their scalings for long contexts, from their definitions, and the
refusals that need no device."""

import ctypes
import math

import numpy as np
import pytest

from zenjpegai_amd import _lib, nn


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (32, 10000.0), (100, 500000.0), (1024, 2.0)])
def test_unscaled(dim, base):
    f, m = nn.rotary_frequencies(dim, base)
    assert m == 1.0 and f.dtype == np.float64
    want = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    assert np.allclose(f, want, rtol=1e-15, atol=0)


def test_linear_squeezes_positions():
    f, m = nn.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert m == 1.0 and np.array_equal(f, nn.rotary_frequencies(64)[0] / 4.0)


@pytest.mark.parametrize("dim", [4, 64, 128])
def test_ntk_divides_the_slowest_alone(dim):
    f, m = nn.rotary_frequencies(dim, scaling="ntk", factor=8.0)
    g, _ = nn.rotary_frequencies(dim)
    assert m == 1.0 and f[0] == 1.0
    assert f[-1] == pytest.approx(g[-1] / 8.0, rel=1e-13)
    assert (f[1:] < g[1:]).all()
    step = f[1:] / f[:-1]
    assert np.allclose(step, step[0], rtol=1e-12, atol=0)


@pytest.mark.parametrize("factor,length", [(1.0, 2048.0), (4.0, 2048.0), (16.0, 100.0)])
def test_yarn_keeps_the_fast_and_divides_the_slow(factor, length):
    f, m = nn.rotary_frequencies(128, scaling="yarn", factor=factor, trained_length=length)
    g, _ = nn.rotary_frequencies(128)
    assert m == np.float32(0.1 * math.log(factor) + 1.0)
    turns = length * g / (2 * math.pi)
    for fi, gi, r in zip(f, g, turns):
        share = 1.0 if r >= 32 else 0.0 if r <= 1 else (r - 1) / 31
        assert fi == pytest.approx(share * gi + (1 - share) * gi / factor, rel=1e-13)
    assert factor == 1.0 or (turns > 32).any() and (turns < 1).any() or length < 201


@pytest.mark.parametrize("dim,args", [
    (0, {}), (3, {}), (-2, {}), (1026, {}),
    (64, {"base": 0.0}), (64, {"base": -1.0}), (64, {"base": float("nan")}), (64, {"base": float("inf")}),
    (64, {"scaling": "linear", "factor": 0.5}), (64, {"scaling": "ntk", "factor": float("nan")}),
    (2, {"scaling": "ntk", "factor": 2.0}),
    (64, {"scaling": "yarn", "factor": 2.0}), (64, {"scaling": "yarn", "factor": 2.0, "trained_length": float("inf")})])
def test_refusals(dim, args):
    with pytest.raises(_lib.HipError) as e:
        nn.rotary_frequencies(dim, **args)
    assert e.value.kind == "InvalidArgument" and "rotary frequencies" in str(e.value)


def test_null_arguments():
    L = _lib.lib()
    f, m = (ctypes.c_double * 32)(), ctypes.c_float()
    assert L.zjai_rotary_frequencies(64, 1e4, 0, 1.0, 0.0, None, ctypes.byref(m)) == _lib.E_INVALID_ARGUMENT
    assert L.zjai_rotary_frequencies(64, 1e4, 0, 1.0, 0.0, f, None) == _lib.E_INVALID_ARGUMENT
    assert L.zjai_rotary_frequencies(64, 1e4, 4, 1.0, 0.0, f, ctypes.byref(m)) == _lib.E_INVALID_ARGUMENT
    for name in ("rotary_noalloc", "causal_conv_noalloc", "causal_conv_step", "selective_scan_noalloc", "selective_scan_step"):
        assert getattr(L, "zjai_" + name)(None, None) == _lib.E_INVALID_ARGUMENT
