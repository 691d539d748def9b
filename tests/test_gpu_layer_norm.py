"""Layer norm, its gradients and clipping by the global norm on encrypted tiles, decrypted, against the formulas in float64.

What the scheme adds is noise: at a scale of 2^42 an encryption is off by less than 2^-30 a slot, a key switch or rescale by less than 2^-33; a row sum of 96 columns, the square of a value up to 4
and the slopes of a polynomial of degree 15 (T_8 has 64, its coefficients fall) make that less than 2^-18.  2^-14 is what products have to meet here, and so does this."""
import ctypes as C

import numpy as np
import pytest
from numpy.polynomial import chebyshev

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -14


@pytest.fixture(scope="module")
def deep(pkg):
    """Tiles of 16 x 32 in a ring with room for a layer norm and its gradients."""
    g = pkg.open_gpu(pkg.make_params(log_n=10, max_level=16, dnum=5, num_special=3, hamming_weight=32))
    g.keygen()
    yield pkg.open_hemmer(g)
    g.close()


def _place(v, lo, hi):
    return (2.0 * v - hi - lo) / (hi - lo)


def _encrypt(h, x, level=None, seed=0):
    """x [column tile][token tile][rows][width] -> one handle, members in that order"""
    import importlib
    pkg = importlib.import_module(type(h).__module__.rsplit(".", 1)[0])
    T, B, rows, w = x.shape
    msgs = np.zeros((T * B, h.lib.slots))
    msgs[:, : rows * w] = x.reshape(T * B, -1)
    return pkg.CtxtTensor(h.lib.encrypt_many(msgs, level or h.lib.L, [seed * 1000 + 17 * k + 1 for k in range(T * B)]), rows, w, w)


def _decrypt(h, t, T, B):
    members = h.lib.ct_meta(t.ct)[2]
    assert members == T * B
    z = h.lib.decrypt_many([(t.ct, k) for k in range(members)])
    imag = np.abs(z.imag).max()
    assert imag < TOL
    return z.real[:, : t.rows * t.width].reshape(T, B, t.rows, t.width)


def _tiles(x, T, w):
    """[B][rows][columns] -> [T][B][rows][w] with zeros behind the columns"""
    B, rows, D = x.shape
    p = np.zeros((B, rows, T * w))
    p[:, :, :D] = x
    return p.reshape(B, rows, T, w).transpose(2, 0, 1, 3)


def _whole(t, D):
    T, B, rows, w = t.shape
    return t.transpose(1, 2, 0, 3).reshape(B, rows, T * w)[:, :, :D]


def _model(x, gamma, beta, eps, rng, c):
    mean = x.mean(-1, keepdims=True)
    var = ((x - mean) ** 2).mean(-1, keepdims=True)
    r = chebyshev.chebval(_place(var + eps, *rng), c)
    xhat = (x - mean) * r
    return xhat * gamma + beta, xhat, r


def _data(rng, B, rows, D):
    x = rng.uniform(-1, 1, (B, rows, D))
    return x * rng.uniform(0.8, 1.6, (B, rows, 1)) + rng.uniform(-0.5, 0.5, (B, rows, 1))   # rows with deviations of 0.4 to 1, and means


RANGE = (0.1, 1.3)
CASES = [  # column tiles, token tiles, columns, degree, weights
    (1, 1, 32, 7, True), (1, 2, 32, 3, False), (1, 1, 20, 7, True), (2, 1, 64, 7, True), (3, 2, 96, 15, True), (3, 1, 70, 15, True), (2, 3, 33, 7, False), (4, 1, 97, 15, False), (3, 2, 96, 7, False),
]


@pytest.mark.parametrize("T,B,D,degree,weights", CASES)
def test_forward_and_backward(deep, T, B, D, degree, weights):
    h, w, rows, eps = deep, 32, 16, 1e-3
    rng = np.random.default_rng(D * 10 + T)
    x, dy = _data(rng, B, rows, D), rng.uniform(-1, 1, (B, rows, D))
    gamma, beta = (rng.uniform(0.5, 1.5, D), rng.uniform(-1, 1, D)) if weights else (None, None)
    g1, b1 = (gamma, beta) if weights else (np.ones(D), np.zeros(D))
    c, depth = h.polynomial("rsqrt", *RANGE, degree)
    y0, xhat0, r0 = _model(x, g1, b1, eps, RANGE, c)
    ct = _encrypt(h, _tiles(x, T, w), seed=1)
    y, xhat, rstd = h.layer_norm(ct, D, RANGE, groups=T, gamma=gamma, beta=beta, eps=eps, degree=degree)
    factor = weights or D < T * w
    assert h.lib.ct_meta(rstd.ct)[0] == h.lib.L - 3 - depth and h.lib.ct_meta(xhat.ct)[0] == h.lib.L - 4 - depth and h.lib.ct_meta(y.ct)[0] == h.lib.L - 4 - depth - factor
    got = _decrypt(h, y, T, B)
    assert np.abs(_whole(got, D) - y0).max() < TOL
    assert np.abs(got.transpose(1, 2, 0, 3).reshape(B, rows, -1)[:, :, D:]).max(initial=0.0) < TOL   # zeros behind the columns
    assert np.abs(_whole(_decrypt(h, xhat, T, B), D) - xhat0).max() < TOL
    assert np.abs(_decrypt(h, rstd, 1, B)[0] - r0).max() < TOL   # in all columns
    # the formulas of the gradients, from the same xhat and rstd
    g = dy * g1
    mean, dot = g.mean(-1, keepdims=True), (g * xhat0).mean(-1, keepdims=True)
    dx0 = r0 * (g - mean - xhat0 * dot)
    dx, dgamma, dbeta = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), seed=2), xhat, rstd, D, groups=T, gamma=gamma)
    got = _decrypt(h, dx, T, B)
    assert np.abs(_whole(got, D) - dx0).max() < TOL
    assert np.abs(got.transpose(1, 2, 0, 3).reshape(B, rows, -1)[:, :, D:]).max(initial=0.0) < TOL
    dg, db = _whole(_decrypt(h, dgamma, T, 1), D), _whole(_decrypt(h, dbeta, T, 1), D)
    total = B * rows   # sums of as many terms, each as exact as a value of the forward pass
    assert np.abs(dg - (dy * xhat0).sum((0, 1))).max() < total * TOL / 8 and np.abs(db - dy.sum((0, 1))).max() < total * TOL / 8
    # and differences of a layer norm with the true root: the polynomial's relative error comes in once by every factor of the root
    v = np.linspace(*RANGE, 2001)
    rel = np.abs(chebyshev.chebval(_place(v, *RANGE), c) * np.sqrt(v) - 1).max()
    step, true = 1e-5, lambda z: (((z - z.mean(-1, keepdims=True)) / np.sqrt(z.var(-1, keepdims=True) + eps) * g1 + b1) * dy).sum()  # noqa: E731
    for b, row, col in [(0, 0, 0), (B - 1, rows - 1, D - 1), (0, 7, D // 2)]:
        up, down = x.copy(), x.copy()
        up[b, row, col] += step
        down[b, row, col] -= step
        want = (true(up) - true(down)) / (2 * step)
        slack = r0[b, row, 0] * (np.abs(g[b, row, col]) + np.abs(mean[b, row, 0]) + np.abs(xhat0[b, row, col] * dot[b, row, 0]))
        assert abs(_whole(got, D)[b, row, col] - want) < TOL + 4 * rel * slack + 1e-6


@pytest.mark.parametrize("lo,hi,degree", [(0.1, 1.3, 7), (0.2, 1.2, 15), (0.2, 0.9, 31), (0.25, 0.75, 31)])
@pytest.mark.parametrize("tokens", [(5, 0), (16, 0), (0, 0), (1, 15)])
def test_rows_that_are_named_as_padding(deep, lo, hi, degree, tokens):
    """Ranges so narrow that the polynomial's terms at a variance of 0 reach 26 to 10^17: the padded rows come out as beta all the same, and the tokens beside them as ever."""
    h, T, B, D, w, rows = deep, 2, 2, 50, 32, 16
    rng = np.random.default_rng(degree)
    x, dy, gamma, beta = rng.uniform(-1, 1, (B, rows, D)), rng.uniform(-1, 1, (B, rows, D)), rng.uniform(0.5, 1.5, D), rng.uniform(-1, 1, D)
    x *= np.sqrt(rng.uniform(lo + 0.05, hi - 0.05, (B, rows, 1))) / x.std(-1, keepdims=True)
    x += rng.uniform(-0.5, 0.5, (B, rows, 1))
    for b, n in enumerate(tokens):
        x[b, n:], dy[b, n:] = 0.0, 0.0
    c, _ = h.polynomial("rsqrt", lo, hi, degree)
    y0, xhat0, r0 = _model(x, gamma, beta, 1e-3, (lo, hi), c)
    for b, n in enumerate(tokens):
        y0[b, n:], xhat0[b, n:], r0[b, n:] = beta, 0.0, chebyshev.chebval(0.0, c)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, (lo, hi), groups=T, gamma=gamma, beta=beta, eps=1e-3, degree=degree, tokens=tokens)
    assert np.abs(_whole(_decrypt(h, y, T, B), D) - y0).max() < TOL
    assert np.abs(_whole(_decrypt(h, xhat, T, B), D) - xhat0).max() < TOL
    assert np.abs(_decrypt(h, rstd, 1, B)[0] - r0).max() < TOL
    if degree == 7:
        g = dy * gamma
        dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
        dx, dgamma, dbeta = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), seed=3), xhat, rstd, D, groups=T, gamma=gamma)
        assert np.abs(_whole(_decrypt(h, dx, T, B), D) - dx0).max() < TOL
        assert np.abs(_whole(_decrypt(h, dgamma, T, 1), D) - (dy * xhat0).sum((0, 1))).max() < B * rows * TOL / 8


def test_rows_of_padding_that_are_not_named(deep):
    """In a wide range the polynomial's value at variance 0 is small; the product with the row's zeros is zero, and what comes out is beta."""
    h, T, B, D, w, rows = deep, 2, 2, 50, 32, 16
    rng = np.random.default_rng(5)
    x, dy, gamma, beta = _data(rng, B, rows, D), rng.uniform(-1, 1, (B, rows, D)), rng.uniform(0.5, 1.5, D), rng.uniform(-1, 1, D)
    x[0, 5:], x[1] = 0.0, 0.0   # a tile that ends early, and one that is empty
    dy[0, 5:], dy[1] = 0.0, 0.0
    c, _ = h.polynomial("rsqrt", *RANGE, 7)
    y0, xhat0, r0 = _model(x, gamma, beta, 1e-3, RANGE, c)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, RANGE, groups=T, gamma=gamma, beta=beta, eps=1e-3, degree=7)
    got = _whole(_decrypt(h, y, T, B), D)
    assert np.abs(got - y0).max() < TOL and np.abs(got[1] - beta).max() < TOL
    dx, dgamma, dbeta = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), seed=3), xhat, rstd, D, groups=T, gamma=gamma)
    assert np.abs(_whole(_decrypt(h, dx, T, B), D)[1]).max() < TOL
    assert np.abs(_whole(_decrypt(h, dgamma, T, 1), D) - (dy * xhat0).sum((0, 1))).max() < B * rows * TOL / 8
    assert np.abs(_whole(_decrypt(h, dbeta, T, 1), D) - dy.sum((0, 1))).max() < B * rows * TOL / 8


@pytest.mark.parametrize("D,weights", [(64, False), (64, True), (50, False)])
def test_the_last_levels(deep, D, weights):
    """From the lowest level that is let through down to level 0, and one level less is refused."""
    h, T, B, w, rows = deep, 2, 1, 32, 16
    rng = np.random.default_rng(8)
    x, dy = _data(rng, B, rows, D), rng.uniform(-1, 1, (B, rows, D))
    gamma = rng.uniform(0.5, 1.5, D) if weights else None
    g1 = gamma if weights else np.ones(D)
    c, depth = h.polynomial("rsqrt", *RANGE, 3)
    least = 4 + depth + (weights or D < 64)
    y0, xhat0, r0 = _model(x, g1, 0.0, 1e-3, RANGE, c)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w), least), D, RANGE, groups=T, gamma=gamma, eps=1e-3, degree=3)
    assert h.lib.ct_meta(y.ct)[0] == 0 and np.abs(_whole(_decrypt(h, y, T, B), D) - y0).max() < TOL
    with pytest.raises(Exception):
        h.layer_norm(_encrypt(h, _tiles(x, T, w), least - 1), D, RANGE, groups=T, gamma=gamma, eps=1e-3, degree=3)
    low = 4 + (weights or D < 64) + (D < 64)
    e_x, e_r = _encrypt(h, _tiles(xhat0, T, w), low, seed=5), _encrypt(h, np.broadcast_to(r0, (B, rows, w))[None].copy(), low, seed=6)
    dx, _, _ = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), low, seed=4), e_x, e_r, D, groups=T, gamma=gamma)
    g = dy * g1
    dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
    assert h.lib.ct_meta(dx.ct)[0] == 0 and np.abs(_whole(_decrypt(h, dx, T, B), D) - dx0).max() < TOL
    with pytest.raises(Exception):
        h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), low - 1, seed=4), e_x, e_r, D, groups=T, gamma=gamma)


@pytest.mark.parametrize("dy_level,r_down", [(16, 0), (9, 0), (7, 0), (16, 4), (7, 5)])
def test_gradients_from_several_levels(deep, dy_level, r_down):
    """dy below what the forward pass kept, and a deviation that has lost levels since: the lowest of them counts."""
    h, T, B, D, w, rows = deep, 2, 1, 50, 32, 16
    rng = np.random.default_rng(6)
    x, dy, gamma = _data(rng, B, rows, D), rng.uniform(-1, 1, (B, rows, D)), rng.uniform(0.5, 1.5, D)
    c, depth = h.polynomial("rsqrt", *RANGE, 3)
    _, xhat0, r0 = _model(x, gamma, np.zeros(D), 1e-3, RANGE, c)
    _, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, RANGE, groups=T, gamma=gamma, eps=1e-3, degree=3)
    rstd.ct = h.lib.level_down(rstd.ct, h.lib.ct_meta(rstd.ct)[0] - r_down)
    dx, dgamma, dbeta = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), dy_level, seed=3), xhat, rstd, D, groups=T, gamma=gamma)
    level = min(dy_level - 1, 16 - 4 - depth)
    assert h.lib.ct_meta(dbeta.ct)[0] == level and h.lib.ct_meta(dgamma.ct)[0] == level - 1 and h.lib.ct_meta(dx.ct)[0] == min(level - 3, 16 - 3 - depth - r_down) - 2
    g = dy * gamma
    dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
    assert np.abs(_whole(_decrypt(h, dx, T, B), D) - dx0).max() < TOL
    assert np.abs(_whole(_decrypt(h, dgamma, T, 1), D) - (dy * xhat0).sum((0, 1))).max() < rows * TOL / 8


@pytest.mark.parametrize("shapes", [[(1, 1)], [(1, 1)] * 5, [(2, 1), (1, 3), (1, 1)], [(5, 6), (1, 1), (30, 1)]])
@pytest.mark.parametrize("norm", [0.7, 2.0, 3.9])
def test_clipping(deep, shapes, norm):
    h, rng, degree = deep, np.random.default_rng(len(shapes)), 15
    xs = [rng.normal(0, 1, (T, B, 16, 32)) for T, B in shapes]
    size = np.sqrt(sum((x ** 2).sum() for x in xs))
    xs = [x * norm / size for x in xs]
    c, depth = h.polynomial("clip", 1.0, 4.0, degree)
    levels = [h.lib.L - k % 3 for k in range(len(xs))]   # gradients of several levels
    grads = [_encrypt(h, x, level, seed=4 + k) for k, (x, level) in enumerate(zip(xs, levels))]
    f = chebyshev.chebval(_place(norm ** 2, 0.0, 16.0), c)
    assert abs(f - min(1.0, 1.0 / norm)) < 0.05
    outs, square = h.clip_grad_norm(grads, 1.0, 4.0, degree)
    assert np.abs(h.lib.decrypt(square) - norm ** 2).max() < 16 * TOL and h.lib.ct_meta(square)[0] == min(levels) - 1
    assert np.abs(h.lib.decrypt(h.grad_norm_squared(grads)) - norm ** 2).max() < 16 * TOL
    for o, x, (T, B) in zip(outs, xs, shapes):
        assert np.abs(_decrypt(h, o, T, B) - x * f).max() < TOL and h.lib.ct_meta(o.ct)[0] == min(levels) - 3 - depth


@pytest.mark.parametrize("degree", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 31])
def test_polynomials_of_every_kind_of_degree(deep, degree):
    """One tensor whose values give the norm that is wanted; degrees whose parts are constants, single terms or empty among them."""
    h, norm = deep, 1.3
    c, depth = h.polynomial("clip", 1.0, 2.0, degree)
    x = np.full((1, 1, 16, 32), norm / np.sqrt(512.0))
    outs, _ = h.clip_grad_norm([_encrypt(h, x)], 1.0, 2.0, degree)
    assert h.lib.ct_meta(outs[0].ct)[0] == h.lib.L - 3 - depth
    assert np.abs(_decrypt(h, outs[0], 1, 1) - x * chebyshev.chebval(_place(norm ** 2, 0.0, 4.0), c)).max() < TOL


def test_a_step_of_training(deep):
    """A product, its layer norm, the gradients back to the weights, and all of them clipped together."""
    h, rng, d = deep, np.random.default_rng(9), 16
    a, b = rng.uniform(-1, 1, (2, d, d)), rng.uniform(-1, 1, (2, d, d))
    gamma, beta, dy = rng.uniform(0.5, 1.5, 2 * d), rng.uniform(-1, 1, 2 * d), rng.uniform(-0.05, 0.05, (1, d, 2 * d))
    prod = h.single_cc_matmul(h.encrypt2(a[0], a[1], nonce=5), h.encrypt2(b[0], b[1], nonce=6), 12)   # two heads side by side
    x = np.concatenate([a[0] @ b[0], a[1] @ b[1]], axis=1)[None]
    wide = type(prod)(prod.ct, d, 2 * d, 2 * d)
    rng_var, eps = (0.2, 6.0), 1e-3
    var = x.var(-1) + eps
    assert rng_var[0] < var.min() and var.max() < rng_var[1]
    c, _ = h.polynomial("rsqrt", *rng_var, 15)
    y0, xhat0, r0 = _model(x, gamma, beta, eps, rng_var, c)
    y, xhat, rstd = h.layer_norm(wide, 2 * d, rng_var, gamma=gamma, beta=beta, eps=eps, degree=15)
    assert np.abs(_whole(_decrypt(h, y, 1, 1), 2 * d) - y0).max() < 4 * TOL   # the product brings an error of its own, up to TOL
    fresh, (hx, hr) = 16, [np.broadcast_to(v, x.shape) for v in (xhat0, r0)]   # (as after a refresh of what the forward pass kept)
    e_dy, e_x, e_r = (_encrypt(h, _tiles(np.ascontiguousarray(v), 1, 2 * d), fresh, seed=20 + k) for k, v in enumerate((dy, hx, hr)))
    dx, dgamma, dbeta = h.layer_norm_backward(e_dy, e_x, e_r, 2 * d, gamma=gamma)
    g = dy * gamma
    dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
    dg0, db0 = (dy * xhat0).sum((0, 1)), dy.sum((0, 1))
    assert np.abs(_whole(_decrypt(h, dx, 1, 1), 2 * d) - dx0).max() < TOL
    # the gradients of the weights stand in all sixteen rows, so they count sixteen times
    norm2 = (dx0 ** 2).sum() + d * ((dg0 ** 2).sum() + (db0 ** 2).sum())
    bound = 4 * np.sqrt(norm2)
    limit = np.sqrt(norm2) / 2
    cc, _ = h.polynomial("clip", limit, bound, 7)
    f = chebyshev.chebval(_place(norm2, 0.0, bound ** 2), cc)
    outs, square = h.clip_grad_norm([dx, dgamma, dbeta], limit, bound, 7)
    assert abs(h.lib.decrypt(square)[0].real - norm2) < 16 * TOL
    for o, v in zip(outs, (dx0[0], np.broadcast_to(dg0, (d, 2 * d)), np.broadcast_to(db0, (d, 2 * d)))):
        assert np.abs(_decrypt(h, o, 1, 1)[0, 0] - v * f).max() < TOL


def test_replayed_from_a_graph(deep):
    """A layer norm without weights, its gradients and their clipping need nothing from the host after their first run."""
    h, T, B, D, w, rows = deep, 2, 1, 64, 32, 16
    rng = np.random.default_rng(11)
    x, dy = [_data(rng, B, rows, D) for _ in range(2)], rng.uniform(-1, 1, (B, rows, D))
    cx, other, cdy = _encrypt(h, _tiles(x[0], T, w)), _encrypt(h, _tiles(x[1], T, w), seed=7), _encrypt(h, _tiles(dy, T, w), seed=8)

    def step():
        y, xhat, rstd = h.layer_norm(cx, D, RANGE, groups=T, degree=3)
        grads = h.layer_norm_backward(cdy, xhat, rstd, D, groups=T)
        square = h.grad_norm_squared([cdy])
        return [y.ct, xhat.ct, rstd.ct, square, *[t.ct for t in grads]], (y, xhat, rstd, grads)

    first = [h.lib.ct_export(o) for o in step()[0]]
    h.lib.graph_begin()
    outs, held = step()
    graph = h.lib.graph_end()
    keep = h.lib.ct_export(cx.ct)
    h.lib.ct_import(cx.ct, h.lib.ct_export(other.ct))
    h.lib.graph_launch(graph)
    c, _ = h.polynomial("rsqrt", *RANGE, 3)
    assert np.abs(_whole(_decrypt(h, held[0], T, B), D) - _model(x[1], 1.0, 0.0, 1e-5, RANGE, c)[0]).max() < TOL
    h.lib.ct_import(cx.ct, keep)
    h.lib.graph_launch(graph)
    for o, want in zip(outs, first):
        assert np.array_equal(h.lib.ct_export(o), want)


def test_ranges_without_end(deep):
    """Masks that depend on the range are kept up to a number; beyond it a call makes its own, with the same result."""
    h, D, w, rows = deep, 32, 32, 16
    rng = np.random.default_rng(12)
    x = _data(rng, 1, rows, D)
    cx = _encrypt(h, _tiles(x, 1, w))

    def used():
        total, now = C.c_uint64(), C.c_uint64()
        h.lib._fn("mem_info")(h.lib.ctx, C.byref(total), C.byref(now))
        return now.value

    sizes = []
    for k in range(140):
        rng_k = (0.1, 1.3 + 0.01 * k)
        y, _, _ = h.layer_norm(cx, D, rng_k, degree=3)
        if k % 35 == 34:
            c, _ = h.polynomial("rsqrt", *rng_k, 3)
            assert np.abs(_whole(_decrypt(h, y, 1, 1), D) - _model(x, 1.0, 0.0, 1e-5, rng_k, c)[0]).max() < TOL
            sizes.append(used())
    assert sizes[-1] == sizes[-2], sizes


def test_refusals(pkg, deep):
    h, rng = deep, np.random.default_rng(1)
    x = _encrypt(h, rng.uniform(-1, 1, (2, 1, 16, 32)))
    low = _encrypt(h, rng.uniform(-1, 1, (2, 1, 16, 32)), 7)
    one = _encrypt(h, rng.uniform(-1, 1, (1, 1, 16, 32)))

    def refused(call, *a, **k):
        with pytest.raises(pkg.HBError) as e:
            call(*a, **k)
        assert e.value.code == -1, e.value

    for columns in (32, 0, -1, 65):
        refused(h.layer_norm, x, columns, RANGE, groups=2)
        refused(h.layer_norm_backward, x, x, one, columns, groups=2)
    for groups in (0, -1, 3):
        refused(h.layer_norm, x, 64, RANGE, groups=groups)
    for bad in ((0.0, 1.0), (1.0, 1.0), (float("nan"), 1.0), (0.1, float("inf"))):
        refused(h.layer_norm, x, 64, bad, groups=2)
    for degree in (0, -3, 64):
        refused(h.layer_norm, x, 64, RANGE, groups=2, degree=degree)
        refused(h.clip_grad_norm, [x], 1.0, 2.0, degree)
    refused(h.layer_norm, x, 64, RANGE, groups=2, tokens=[17])
    refused(h.layer_norm, x, 64, RANGE, groups=2, tokens=[-1])
    for tokens in ([], [1, 2]):
        with pytest.raises(ValueError):
            h.layer_norm(x, 64, RANGE, groups=2, tokens=tokens)
    refused(h.layer_norm, x, 64, RANGE, groups=2, eps=-1.0)
    refused(h.layer_norm, x, 64, RANGE, groups=2, eps=float("nan"))
    refused(h.layer_norm, x, 64, RANGE, groups=2, gamma=np.full(64, np.inf))
    refused(h.layer_norm_backward, x, x, one, 64, groups=2, gamma=np.full(64, np.nan))
    refused(h.layer_norm, low, 64, RANGE, groups=2, degree=7)
    refused(h.layer_norm_backward, x, x, x, 64, groups=2)   # a deviation per member of a column tile
    refused(h.layer_norm_backward, x, one, one, 64, groups=2)
    refused(h.layer_norm, pkg.CtxtTensor(x.ct, 16, 16, 16), 32, RANGE, groups=2)   # tiles that do not fill the slots
    refused(h.layer_norm, pkg.CtxtTensor(x.ct, 16, 24, 24), 48, RANGE, groups=2)
    refused(h.layer_norm, pkg.CtxtTensor(x.ct, 2 ** 30, 2 ** 30, 2 ** 30), 48, RANGE, groups=2)
    refused(h.clip_grad_norm, [x], 2.0, 2.0, 7)
    refused(h.clip_grad_norm, [x], -1.0, 2.0, 7)
    refused(h.clip_grad_norm, [x, _encrypt(h, rng.uniform(-1, 1, (1, 1, 16, 32)), 6)], 1.0, 2.0, 7)
    refused(h.clip_grad_norm, [], 1.0, 2.0)
    refused(h.grad_norm_squared, [])
    refused(h.grad_norm_squared, [_encrypt(h, rng.uniform(-1, 1, (1, 1, 16, 32)), 0 + 1), type(x)(h.lib.level_down(one.ct, 0), 16, 32, 32)])
    null = (C.c_void_p * 2)()
    assert h._fn("grad_norm_squared")(h.h, null, 2, C.byref(C.c_void_p())) == -1
    assert h._fn("clip_grad_norm")(h.h, null, 2, C.c_double(1.0), C.c_double(2.0), 7, null, None) == -1
    assert h._fn("layer_norm")(h.h, x.ct.ptr, 16, 32, 32, 2, 64, None, None, C.c_double(0.0), C.c_double(0.1), C.c_double(1.0), 7, None, None, None, None) == -1


def test_the_full_ring(pkg, gpu_full):
    """128 tokens of 768 columns at the benchmark's parameters, forward with weights, and the gradients of what it kept."""
    h = pkg.open_hemmer(gpu_full)
    T, B, D, w, rows = 3, 1, 768, 256, 128
    rng = np.random.default_rng(7)
    x, dy, gamma, beta = _data(rng, B, rows, D), rng.uniform(-1, 1, (B, rows, D)), rng.uniform(0.5, 1.5, D), rng.uniform(-1, 1, D)
    c, depth = h.polynomial("rsqrt", *RANGE, 7)
    y0, xhat0, r0 = _model(x, gamma, beta, 1e-5, RANGE, c)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, RANGE, groups=T, gamma=gamma, beta=beta, degree=7)
    assert np.abs(_whole(_decrypt(h, y, T, B), D) - y0).max() < TOL
    e_x, e_r = _encrypt(h, _tiles(xhat0, T, w), 8, seed=8), _encrypt(h, np.broadcast_to(r0, (B, rows, w))[None].copy(), 8, seed=9)   # as after a refresh
    dx, dgamma, dbeta = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), seed=3), e_x, e_r, D, groups=T, gamma=gamma)
    g = dy * gamma
    dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
    assert np.abs(_whole(_decrypt(h, dx, T, B), D) - dx0).max() < TOL
    assert np.abs(_whole(_decrypt(h, dgamma, T, 1), D) - (dy * xhat0).sum((0, 1))).max() < rows * TOL / 8
    assert np.abs(_whole(_decrypt(h, dbeta, T, 1), D) - dy.sum((0, 1))).max() < rows * TOL / 8
    h.close()
