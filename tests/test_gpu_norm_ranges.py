"""Layer norms of values of any size.

The mask that brings a row's sum of squares to the polynomial's range holds 2 / ((hi - lo) columns), whose rounding, half a unit of 2^-42 a coefficient, is 2 units a slot
(32 columns: 64 coefficients that are not zero) and some 13 in a sum of the 32 copies of a row: 2e-4 of 7.6e4 units for a range a million wide and 96 columns, and ten times that where a
neighbour's variance is as many times larger.  Variances are squares, so a root's relative error is half of theirs; 2^-14 is what has to be met."""
import numpy as np
import pytest

from test_gpu_layer_norm import TOL, _data, _decrypt, _encrypt, _model, _tiles, _whole, deep  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1.0, 30.0, 1e3, 3e3])
@pytest.mark.parametrize("T,B,D,tokens", [(3, 2, 96, None), (3, 1, 70, None), (2, 2, 64, (16, 5))])
def test_values_of_a_size(deep, T, B, D, tokens, size):  # noqa: F811
    h, w, rows, degree = deep, 32, 16, 7
    rng = np.random.default_rng(D)
    x = _data(rng, B, rows, D) * size
    for b, n in enumerate(tokens or ()):
        x[b, n:] = 0.0
    gamma, beta = rng.uniform(0.5, 1.5, D), rng.uniform(-1, 1, D)
    span, eps = (0.1 * size ** 2, 1.3 * size ** 2), 1e-3 * size ** 2
    c, depth = h.polynomial("rsqrt", *span, degree)
    y0, xhat0, r0 = _model(x, gamma, beta, eps, span, c)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, span, groups=T, gamma=gamma, beta=beta, eps=eps, degree=degree, tokens=tokens)
    assert h.lib.ct_meta(rstd.ct)[0] == h.lib.L - 3 - depth and h.lib.ct_meta(xhat.ct)[0] == h.lib.L - 4 - depth and h.lib.ct_meta(y.ct)[0] == h.lib.L - 5 - depth
    live = np.ones((B, rows), bool)
    for b, n in enumerate(tokens or ()):
        live[b, n:] = False
    got_y, got_x, got_r = _whole(_decrypt(h, y, T, B), D), _whole(_decrypt(h, xhat, T, B), D), _decrypt(h, rstd, 1, B)[0]
    assert np.abs(got_y - y0)[live].max() < TOL and np.abs(got_x - xhat0)[live].max() < TOL
    assert np.abs(got_r / r0 - 1)[live].max() < TOL
    assert np.abs(got_y - beta)[~live].max(initial=0.0) < TOL


@pytest.mark.parametrize("width", [1e21, 1e40, 1e308])
def test_ranges_that_are_refused(pkg, deep, width):  # noqa: F811
    """64 columns: both masks have the same number of units at ((2 / 64 / width) / 64^2)^(1/3) 2^42, which is 2^16 for a width of 2^61."""
    h = deep
    x = _encrypt(h, np.random.default_rng(1).uniform(-1, 1, (2, 1, 16, 32)))
    with pytest.raises(pkg.HBError) as e:
        h.layer_norm(x, 64, (0.1, width), groups=2, degree=3)
    assert e.value.code == -1 and "range" in str(e.value)


def test_the_full_ring(pkg, gpu_full):
    """768 columns, values of some hundreds: 1e5 units for a mask without the shift."""
    h = pkg.open_hemmer(gpu_full)
    T, B, D, w, rows, size = 3, 1, 768, 256, 128, 300.0
    rng = np.random.default_rng(7)
    x, span, eps = _data(rng, B, rows, D) * size, (0.1 * size ** 2, 1.3 * size ** 2), 1e-3 * size ** 2
    c, depth = h.polynomial("rsqrt", *span, 7)
    y0, _, r0 = _model(x, 1.0, 0.0, eps, span, c)
    y, _, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, span, groups=T, eps=eps, degree=7)
    assert h.lib.ct_meta(y.ct)[0] == h.lib.L - 4 - depth
    assert np.abs(_whole(_decrypt(h, y, T, B), D) - y0).max() < TOL and np.abs(_decrypt(h, rstd, 1, B)[0] / r0 - 1).max() < TOL
    h.close()


def test_recorded(deep):  # noqa: F811
    """A layer norm in a wide range, whose x is shrunk, as a graph on other values."""
    h, T, B, D, w, rows, size = deep, 2, 1, 60, 32, 16, 1e3
    xs = [_data(np.random.default_rng(k), B, rows, D) * size for k in range(2)]
    span = (0.1 * size ** 2, 1.3 * size ** 2)
    c, _ = h.polynomial("rsqrt", *span, 3)
    cx, other = (_encrypt(h, _tiles(x, T, w), seed=k) for k, x in enumerate(xs))
    h.layer_norm(cx, D, span, groups=T, degree=3)
    h.lib.graph_begin()
    y, xhat, rstd = h.layer_norm(cx, D, span, groups=T, degree=3)
    graph = h.lib.graph_end()
    h.lib.graph_launch(graph)
    assert np.abs(_whole(_decrypt(h, y, T, B), D) - _model(xs[0], 1.0, 0.0, 1e-5, span, c)[0]).max() < TOL
    h.lib.ct_import(cx.ct, h.lib.ct_export(other.ct))
    h.lib.graph_launch(graph)
    assert np.abs(_whole(_decrypt(h, y, T, B), D) - _model(xs[1], 1.0, 0.0, 1e-5, span, c)[0]).max() < TOL
