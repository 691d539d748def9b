"""The polynomials of layer_norm and clip_grad_norm, which need no device, and what the Python layer checks of its arguments."""
import ctypes as C
import os
import subprocess
from types import SimpleNamespace

import numpy as np
import pytest
from numpy.polynomial import chebyshev

from conftest import PKG_NAME, ROOT


@pytest.fixture(scope="module")
def polynomial(pkg):
    C.CDLL(pkg.CUDA_LIB, mode=C.RTLD_GLOBAL)
    h = object.__new__(pkg.Hemmer)
    h.dll, h.prefix = C.CDLL(pkg.HELLM_LIB), "hb_hemmer_"
    return h.polynomial


def _depth(n):
    """Levels by following what is multiplied with what: (level of T_m, then of a sum of T_1 .. T_n)"""
    if n <= 3:
        return n
    m = 1 << (n.bit_length() - 1)
    high, low = (_depth(n - m) if n > m else 0), _depth(m - 1)
    return max(max(m.bit_length() - 1, high) + 1, low)


@pytest.mark.parametrize("degree", [1, 2, 3, 4, 5, 7, 8, 15, 16, 22, 31, 63])
@pytest.mark.parametrize("lo,hi", [(0.25, 4.0), (1e-3, 2e-3), (0.5, 50.0)])
def test_inverse_root(polynomial, degree, lo, hi):
    c, depth = polynomial("rsqrt", lo, hi, degree)
    want = chebyshev.chebinterpolate(lambda u: 1.0 / np.sqrt(0.5 * (hi + lo) + 0.5 * (hi - lo) * u), degree)
    assert np.abs(c - want).max() < 1e-12 / np.sqrt(lo) and depth == _depth(degree)
    # interpolation of 1 / sqrt: the error falls by rho a degree, rho = (sqrt k + 1) / (sqrt k - 1), k = hi / lo
    rho = (np.sqrt(hi / lo) + 1) / (np.sqrt(hi / lo) - 1)
    u = np.linspace(-1, 1, 1001)
    err = np.abs(chebyshev.chebval(u, c) * np.sqrt(0.5 * (hi + lo) + 0.5 * (hi - lo) * u) - 1).max()
    assert err < 20 * np.sqrt(hi / lo) * rho ** -degree + 1e-11


@pytest.mark.parametrize("degree", [1, 3, 7, 15, 31, 63])
def test_clip(polynomial, degree):
    c, depth = polynomial("clip", 1.0, 4.0, degree)
    f = lambda s: np.where(s > 1.0, 1.0 / np.sqrt(np.maximum(s, 1.0)), 1.0)  # noqa: E731
    assert np.abs(c - chebyshev.chebinterpolate(lambda u: f(8.0 * (u + 1.0)), degree)).max() < 1e-12 and depth == _depth(degree)
    u = np.linspace(-1, 1, 2001)
    err = np.abs(chebyshev.chebval(u, c) - f(8.0 * (u + 1.0))).max()
    assert err < {1: 0.6, 3: 0.3, 7: 0.13, 15: 0.05, 31: 0.03, 63: 0.015}[degree]   # a kink: the error falls like 1 / degree


def test_polynomials_that_are_refused(pkg, polynomial):
    for which, a, b, degree in (("rsqrt", 0.0, 1.0, 7), ("rsqrt", -1.0, 1.0, 7), ("rsqrt", 1.0, 1.0, 7), ("rsqrt", 2.0, 1.0, 7), ("rsqrt", float("nan"), 1.0, 7), ("rsqrt", 1.0, float("inf"), 7),
                                ("rsqrt", 1.0, float("nan"), 7), ("rsqrt", 1.0, 2.0, 0), ("rsqrt", 1.0, 2.0, 64), ("rsqrt", 1.0, 2.0, -1), ("clip", 0.0, 1.0, 7), ("clip", 1.0, 1.0, 7), ("clip", 2.0, 1.0, 7),
                                ("clip", 1.0, float("inf"), 7), ("clip", float("nan"), 2.0, 7), ("clip", 1.0, 1e200, 7), ("clip", 1e-200, 1e-190, 7)):
        with pytest.raises(pkg.HBError) as e:
            polynomial(which, a, b, degree)
        assert e.value.code == -1


def test_rules_of_dispatch(tmp_path):
    exe = str(tmp_path / "norm_rules")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "integration", "norm_rules.cpp"), "-I", os.path.join(ROOT, PKG_NAME, "csrc"), "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout[:2000]


def test_lists_of_another_length(pkg):
    """Plaintexts that are not one per column tile, and weights that are not one per column, do not reach the library."""
    lib = object.__new__(pkg.capi.Lib)
    lib.alive = False
    x = SimpleNamespace(ptr=None)
    for lists in ({"gamma": [x]}, {"beta": [x] * 3}, {"gamma": [x] * 2, "beta": [x]}):
        with pytest.raises(ValueError):
            lib.norm_affine(x, 2, **lists)
    with pytest.raises(ValueError):
        lib.norm_affine(x, 2 ** 31, gamma=[x])
    h = object.__new__(pkg.Hemmer)
    h._call = lambda *a, **k: pytest.fail("reached the library")
    h.lib = SimpleNamespace(ct_meta=lambda ct: (3, 2, 6, 1))
    t = pkg.CtxtTensor(x, 16, 16, 32)
    for tokens in ([], [1, 2], [1, 2, 3, 4], [2 ** 31] * 3):
        with pytest.raises(ValueError):
            h.layer_norm(t, 40, (1.0, 2.0), groups=2, tokens=tokens)
    for gamma in (np.ones(39), np.ones(41), np.ones((40, 1)), 1.0):
        with pytest.raises(ValueError):
            h.layer_norm(t, 40, (1.0, 2.0), groups=2, gamma=gamma)
        with pytest.raises(ValueError):
            h.layer_norm_backward(t, t, t, 40, groups=2, gamma=gamma)
