"""The global norm of gradients that hold their values several times: each counts once.  Bounds as in the tests of the layer norm: 2^-14 of what a slot holds."""
import ctypes as C

import numpy as np
import pytest
from numpy.polynomial import chebyshev

from test_gpu_layer_norm import RANGE, TOL, _data, _decrypt, _encrypt, _model, _place, _tiles, _whole, deep  # noqa: F401

pytestmark = pytest.mark.gpu


def _periodic(rng, members, period):
    return np.tile(rng.uniform(-1, 1, (members, period)), (1, 512 // period)).reshape(1, members, 16, 32)


@pytest.mark.parametrize("periods", [[512], [32], [1], [512, 32], [32, 512], [32, 32, 512, 32], [1, 512], [16, 32, 512, 64], [256, 2, 1], [512, 512], [32, 1, 32]])
def test_every_value_counts_once(deep, periods):  # noqa: F811
    h, rng = deep, np.random.default_rng(sum(periods))
    xs = [_periodic(rng, 1 + k % 3, p) for k, p in enumerate(periods)]
    parts = [(x ** 2).sum() * p / 512 for x, p in zip(xs, periods)]
    size = np.sqrt(sum(parts))
    xs = [x / size * 1.7 for x in xs]
    grads = [_encrypt(h, x, h.lib.L - k % 2, seed=k) for k, x in enumerate(xs)]
    want = 1.7 ** 2
    square = h.grad_norm_squared(grads, periods)
    assert h.lib.ct_meta(square)[0] == min(h.lib.L - k % 2 for k in range(len(xs))) - 1
    assert np.abs(h.lib.decrypt(square) - want).max() < 16 * TOL   # in every slot
    c, _ = h.polynomial("clip", 1.0, 4.0, 7)
    f = chebyshev.chebval(_place(want, 0.0, 16.0), c)
    outs, again = h.clip_grad_norm(grads, 1.0, 4.0, 7, periods=periods)
    assert np.abs(h.lib.decrypt(again) - want).max() < 16 * TOL
    for o, x in zip(outs, xs):
        assert np.abs(_decrypt(h, o, 1, x.shape[1]) - x * f).max() < TOL


def test_without_periods(deep):  # noqa: F811
    """None, a list of none, and periods of all slots are the call without them, bit for bit."""
    h, rng = deep, np.random.default_rng(3)
    grads = [_encrypt(h, rng.uniform(-0.05, 0.05, (1, 2, 16, 32)), seed=k) for k in range(2)]
    want = h.lib.ct_export(h.grad_norm_squared(grads))
    for periods in (None, [None, None], [512, None]):
        assert np.array_equal(h.lib.ct_export(h.grad_norm_squared(grads, periods)), want)
    out = C.c_void_p()
    arr = (C.c_void_p * 2)(*[g.ct.ptr.value for g in grads])
    assert h._fn("grad_norm_squared")(h.h, arr, 2, C.byref(out)) == 0
    assert np.array_equal(h.lib.ct_export(type(grads[0].ct)(h.lib, out, "ct")), want)


def test_gradients_of_a_layer_norm(deep):  # noqa: F811
    """dx, dgamma and dbeta as the framework makes them, clipped by the norm that counts each parameter once."""
    h, T, B, D, w, rows = deep, 2, 2, 50, 32, 16
    rng = np.random.default_rng(6)
    x, dy, gamma = _data(rng, B, rows, D), rng.uniform(-0.1, 0.1, (B, rows, D)), rng.uniform(0.5, 1.5, D)
    c, _ = h.polynomial("rsqrt", *RANGE, 3)
    _, xhat0, r0 = _model(x, gamma, np.zeros(D), 1e-3, RANGE, c)
    e_x, e_r = _encrypt(h, _tiles(xhat0, T, w), 16, seed=5), _encrypt(h, np.broadcast_to(r0, (B, rows, w))[None].copy(), 16, seed=6)
    grads = list(h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), seed=3), e_x, e_r, D, groups=T, gamma=gamma))
    g = dy * gamma
    dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
    dg0, db0 = (dy * xhat0).sum((0, 1)), dy.sum((0, 1))
    norm2 = (dx0 ** 2).sum() + (dg0 ** 2).sum() + (db0 ** 2).sum()
    limit, bound = np.sqrt(norm2) / 2, 2 * np.sqrt(norm2)
    cc, _ = h.polynomial("clip", limit, bound, 7)
    f = chebyshev.chebval(_place(norm2, 0.0, bound ** 2), cc)
    outs, square = h.clip_grad_norm(grads, limit, bound, 7, periods=[None, w, w])
    assert np.abs(h.lib.decrypt(square) - norm2).max() < 16 * TOL * max(1.0, norm2)
    assert np.abs(_whole(_decrypt(h, outs[0], T, B), D) - dx0 * f).max() < TOL
    for o, v in ((outs[1], dg0), (outs[2], db0)):
        assert np.abs(_whole(_decrypt(h, o, T, 1), D) - v * f).max() < B * rows * TOL / 8


def test_periods_that_are_refused(pkg, deep):  # noqa: F811
    h = deep
    x = _encrypt(h, np.random.default_rng(1).uniform(-0.01, 0.01, (1, 1, 16, 32)))
    for p in (0, -1, -32, 3, 33, 1024, 2 ** 30, 2 ** 31 - 1):
        for call in (lambda: h.grad_norm_squared([x, x], [512, p]), lambda: h.clip_grad_norm([x, x], 1.0, 2.0, 7, periods=[p, 512])):
            with pytest.raises(pkg.HBError) as e:
                call()
            assert e.value.code == -1
    with pytest.raises(pkg.HBError):
        h.grad_norm_squared([], [])


def test_recorded(deep):  # noqa: F811
    h, rng = deep, np.random.default_rng(4)
    grads = [_encrypt(h, _periodic(rng, 1, p) / 40, seed=p) for p in (512, 32, 32)]
    want = h.lib.ct_export(h.grad_norm_squared(grads, [512, 32, 32]))
    h.lib.graph_begin()
    out = h.grad_norm_squared(grads, [512, 32, 32])
    graph = h.lib.graph_end()
    h.lib.graph_launch(graph)
    assert np.array_equal(h.lib.ct_export(out), want)
