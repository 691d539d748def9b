"""hb_norm_*, hb_square_sum_many and hb_scale_many against sums of products of Python's own integers, member by member.  All results are whole numbers:
equal or wrong."""
import ctypes as C

import numpy as np
import pytest

from conftest import open_oracle, rand_ct_residues
from test_gpu_tile_products import _ct, _points, _pt, _rand

pytestmark = pytest.mark.gpu


def _primes(g, n):
    return np.array([int(q) for q in g.primes[:n]], dtype=object)[:, None]


def _pair(x, y):
    return np.stack([x[0] * y[0], x[0] * y[1] + x[1] * y[0], x[1] * y[1]])


def _check(g, handle, expected, at, level, polys, scale_pow):
    assert g.ct_meta(handle) == (level, polys, len(expected), scale_pow)
    got = g.ct_export(handle)[..., at].astype(object)
    want = np.stack([e % _primes(g, level + 1) for e in expected])
    assert np.array_equal(got, want)


def _objects(res, at):
    return res[..., at].astype(object)


def _scale(g, level):
    return int(np.rint(g.scales[level]))


SHAPES = [  # column tiles, token tiles, level
    (1, 1, 3), (2, 1, 0), (3, 2, 5), (4, 3, 2), (5, 1, 1), (6, 4, 3), (7, 5, 2), (8, 1, 8), (9, 2, 1), (12, 3, 3), (13, 2, 2), (1, 17, 1), (33, 1, 2), (2, 40, 1), (130, 1, 0),
    (4, 1, 3), (6, 1, 2), (7, 1, 4), (4, 2, 1), (2, 4, 3), (1, 8, 2),
]


@pytest.fixture(params=["small", "mid"])
def ring(request, gpu_small, gpu_mid):
    return gpu_small if request.param == "small" else gpu_mid


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("T,B,level", SHAPES)
def test_squares(ring, T, B, level, edge):
    g = ring
    x, mean = _rand(g, level, T * B, 1, edge=edge), _rand(g, level, B, 2)
    if edge:  # differences as large as they get, of either sign
        mean[::2] = 0
        mean[1::2] = x[0]
        x[: B // 2] = 0
    at = _points(g, np.random.default_rng(T * 100 + B), 12)
    xo, mo = _objects(x, at), _objects(mean, at)
    cx, cm = _ct(g, x), _ct(g, mean)
    for pad in (0, 1, g.slots):
        want = [sum(_pair(xo[t * B + b] - mo[b], xo[t * B + b] - mo[b]) for t in range(T)) - pad * _pair(mo[b], mo[b]) for b in range(B)]
        _check(g, g.norm_squares(cx, T, mean=cm, pad=pad), want, at, level, 3, 2)
    _check(g, g.norm_squares(cx, T), [sum(_pair(xo[t * B + b], xo[t * B + b]) for t in range(T)) for b in range(B)], at, level, 3, 2)


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("T,B,level", SHAPES)
def test_scale(ring, T, B, level, edge):
    g = ring
    x, mean, r, rr = _rand(g, level, T * B, 1, edge=edge), _rand(g, level, B, 2), _rand(g, level, B, 3, edge=edge), _rand(g, level, T * B, 4)
    if edge:
        mean[::2] = 0
        x[: B // 2] = 0
    at = _points(g, np.random.default_rng(T * 100 + B), 12)
    xo, mo, ro, rro = (_objects(v, at) for v in (x, mean, r, rr))
    cx, cm, cr, crr = (_ct(g, v) for v in (x, mean, r, rr))
    of = [(k, k % B) for k in range(T * B)]
    _check(g, g.norm_scale(cx, cr, T, mean=cm), [_pair(xo[k] - mo[b], ro[b]) for k, b in of], at, level, 3, 2)
    _check(g, g.norm_scale(cx, cr, T), [_pair(xo[k], ro[b]) for k, b in of], at, level, 3, 2)
    _check(g, g.norm_scale(cx, crr, T, mean=cm), [_pair(xo[k] - mo[b], rro[k]) for k, b in of], at, level, 3, 2)


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("T,B,level", SHAPES)
def test_affine(ring, T, B, level, edge):
    g = ring
    x = _rand(g, level, T * B, 1, edge=edge)
    gamma, beta = (_rand(g, level, T, s, polys=1, edge=edge)[:, 0] for s in (2, 3))
    at = _points(g, np.random.default_rng(T * 100 + B), 12)
    xo, go, bo = (_objects(v, at) for v in (x, gamma, beta))
    cx, pg, pb, K = _ct(g, x), [_pt(g, v) for v in gamma], [_pt(g, v) for v in beta], _scale(g, level)
    of = [(k, k // B) for k in range(T * B)]
    _check(g, g.norm_affine(cx, T, gamma=pg, beta=pb), [np.stack([xo[k][0] * go[t] + K * bo[t], xo[k][1] * go[t]]) for k, t in of], at, level, 2, 2)
    _check(g, g.norm_affine(cx, T, gamma=pg), [np.stack([xo[k][0] * go[t], xo[k][1] * go[t]]) for k, t in of], at, level, 2, 2)
    _check(g, g.norm_affine(cx, T, beta=pb), [np.stack([xo[k][0] + bo[t], xo[k][1]]) for k, t in of], at, level, 2, 1)


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("T,B,level", SHAPES)
def test_grad_sums(ring, T, B, level, edge):
    g = ring
    dy, gg, xh = (_rand(g, level, T * B, s, edge=edge) for s in (1, 2, 3))
    at = _points(g, np.random.default_rng(T * 100 + B), 12)
    do, go, xo = (_objects(v, at) for v in (dy, gg, xh))
    cd, cg, cx = (_ct(g, v) for v in (dy, gg, xh))
    for handle, y in ((cg, go), (None, do)):
        got = g.norm_grad_sums(cd, cx, T, g=handle)
        _check(g, got[0], [sum(_pair(y[t * B + b], xo[t * B + b]) for t in range(T)) for b in range(B)], at, level, 3, 2)
        _check(g, got[1], [sum(y[t * B + b] for t in range(T)) for b in range(B)], at, level, 2, 1)
        _check(g, got[2], [sum(_pair(do[t * B + b], xo[t * B + b]) for b in range(B)) for t in range(T)], at, level, 3, 2)
        _check(g, got[3], [sum(do[t * B + b] for b in range(B)) for t in range(T)], at, level, 2, 1)


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("T,B,level", SHAPES)
def test_grad_input(ring, T, B, level, edge):
    g = ring
    gg, xh, mean, dot = _rand(g, level, T * B, 1, edge=edge), _rand(g, level, T * B, 2, edge=edge), _rand(g, level, B, 3), _rand(g, level, B, 4, edge=edge)
    if edge:  # the largest differences, and factors of nothing
        mean[::2] = 0
        xh[: B // 2] = 0
    at = _points(g, np.random.default_rng(T * 100 + B), 12)
    go, xo, mo, ao = (_objects(v, at) for v in (gg, xh, mean, dot))
    K, nothing = _scale(g, level), 0 * go[0][:1]
    want = [np.concatenate([K * (go[k] - mo[k % B]), nothing]) - _pair(xo[k], ao[k % B]) for k in range(T * B)]
    _check(g, g.norm_grad_input(*(_ct(g, v) for v in (gg, mean, xh, dot)), T), want, at, level, 3, 2)


LISTS = [[1], [3], [1, 1], [1] * 7, [2, 5, 1], [1, 4, 1, 9, 2], [31, 2], [64], [130, 126], [255, 2], [257], [1] * 40 + [100] * 5]


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{sum(s)}")
def test_square_sum_many(ring, sizes, edge):
    g, level = ring, 2 if sum(sizes) < 100 else 1
    xs = [_rand(g, level, m, 10 + k, edge=edge) for k, m in enumerate(sizes)]
    at = _points(g, np.random.default_rng(len(sizes)), 12)
    want = sum(_pair(m, m) for x in xs for m in _objects(x, at))
    handles = [_ct(g, x) for x in xs]
    _check(g, g.square_sum_many(handles), [want], at, level, 3, 2)
    _check(g, g.square_sum_many(handles + handles[:1]), [want + sum(_pair(m, m) for m in _objects(xs[0], at))], at, level, 3, 2)   # the same handle twice


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{sum(s)}")
def test_scale_many(ring, sizes, edge):
    g, level = ring, 2 if sum(sizes) < 100 else 1
    xs, f = [_rand(g, level, m, 10 + k, edge=edge) for k, m in enumerate(sizes)], _rand(g, level, 1, 9, edge=edge)
    at = _points(g, np.random.default_rng(len(sizes)), 12)
    handles, cf, fo = [_ct(g, x) for x in xs], _ct(g, f), _objects(f, at)[0]
    got = g.scale_many(handles + handles[:1] + [cf], cf)   # the same handle twice, and the factor itself
    assert len(got) == len(xs) + 2
    for h, x in zip(got, xs + xs[:1] + [f]):
        _check(g, h, [_pair(m, fo) for m in _objects(x, at)], at, level, 3, 2)
    _check(g, cf, _objects(f, at), at, level, 2, 1)


def _all_sums(g, level, T, B, at, check_input=True):
    x, z, mean, r = _rand(g, level, T * B, 1, edge=True), _rand(g, level, T * B, 4, edge=True), _rand(g, level, B, 2), _rand(g, level, B, 3, edge=True)
    mean[0] = 0
    xo, zo, mo, ro = (_objects(v, at) for v in (x, z, mean, r))
    cx, cz, cm, cr = (_ct(g, v) for v in (x, z, mean, r))
    _check(g, g.norm_squares(cx, T, mean=cm, pad=7), [sum(_pair(xo[t * B + b] - mo[b], xo[t * B + b] - mo[b]) for t in range(T)) - 7 * _pair(mo[b], mo[b]) for b in range(B)], at, level, 3, 2)
    _check(g, g.norm_scale(cx, cr, T, mean=cm), [_pair(xo[k] - mo[k % B], ro[k % B]) for k in range(T * B)], at, level, 3, 2)
    for handle, q in ((None, xo), (cz, zo)):
        rows, rowsum, cols, colsum = g.norm_grad_sums(cx, cx, T, g=handle)
        _check(g, rows, [sum(_pair(q[t * B + b], xo[t * B + b]) for t in range(T)) for b in range(B)], at, level, 3, 2)
        _check(g, rowsum, [sum(q[t * B + b] for t in range(T)) for b in range(B)], at, level, 2, 1)
        _check(g, cols, [sum(_pair(xo[t * B + b], xo[t * B + b]) for b in range(B)) for t in range(T)], at, level, 3, 2)
        _check(g, colsum, [sum(xo[t * B + b] for b in range(B)) for t in range(T)], at, level, 2, 1)
    K, nothing = _scale(g, level), 0 * xo[0][:1]
    _check(g, g.norm_grad_input(cx, cm, cx, cr, T), [np.concatenate([K * (xo[k] - mo[k % B]), nothing]) - _pair(xo[k], ro[k % B]) for k in range(T * B)], at, level, 3, 2)
    _check(g, g.square_sum_many([cx, cm]), [sum(_pair(v, v) for v in [*xo, *mo])], at, level, 3, 2)


@pytest.mark.parametrize("n_bits", [58, 50, 45, 44, 43])
@pytest.mark.parametrize("T,B", [(19, 2), (8, 1), (5, 1), (2, 9)])
def test_primes_of_other_lengths(pkg, n_bits, T, B):
    """Scaling primes that leave room for eight products of a sum, and those that go by pieces."""
    g = pkg.open_gpu(pkg.make_params(log_n=10, max_level=4, dnum=3 if n_bits < 50 else 5, num_special=3, q0_bits=60, q_bits=n_bits, p_bits=60, hamming_weight=32))
    try:
        _all_sums(g, 3, T, B, np.arange(g.N))
    finally:
        g.close()


@pytest.mark.parametrize("n_bits", [50, 44])
def test_primes_of_other_lengths_in_the_full_ring(pkg, n_bits):
    """Sums of both directions in one kernel, past every reduction."""
    g = pkg.open_gpu(pkg.make_params(log_n=16, max_level=3, dnum=3 if n_bits < 50 else 4, num_special=3, q0_bits=60, q_bits=n_bits, p_bits=60, hamming_weight=32))
    try:
        at = np.array([0, 1, 127, 128, 511, 512, 40000, 65535])
        _all_sums(g, 1, 3, 19, at)
        _all_sums(g, 2, 8, 2, at)
    finally:
        g.close()


def _whole(v, scale):
    return int(np.rint(v * scale))


@pytest.mark.parametrize("edge", [False, True])
@pytest.mark.parametrize("terms,members,polys,level", [(1, 1, 2, 3), (2, 3, 2, 0), (3, 2, 3, 5), (8, 1, 2, 1), (9, 2, 1, 2), (16, 5, 2, 8)])
def test_combine(ring, terms, members, polys, level, edge):
    g = ring
    rng = np.random.default_rng(terms)
    xs = [_rand(g, level, members, 20 + j, polys=polys, edge=edge) for j in range(terms)]
    at = _points(g, rng, 12)
    handles, scale = [_ct(g, x) for x in xs], float(g.scales[level])
    coefficients = [float(v) for v in rng.uniform(-3, 3, terms)]
    coefficients[0] = 0.0 if edge else -1.0
    for constant in (0.0, 0.75, -1234.5):
        k, k0 = [_whole(v, scale) for v in coefficients], _whole(constant, scale) * _scale(g, level)
        want = []
        for b in range(members):
            total = sum(kk * _objects(x, at)[b] for kk, x in zip(k, xs))
            total[0] = total[0] + k0
            want.append(total)
        _check(g, g.combine(handles, coefficients, constant), want, at, level, polys, 2)
        want = [_objects(xs[0], at)[b].copy() for b in range(members)]
        for v in want:
            v[0] = v[0] + _whole(constant, scale)
        _check(g, g.add_const(handles[0], constant), want, at, level, polys, 1)


def test_constants_are_what_encoded_ones_are(gpu_small):
    """Slots of x + v, and of sums with coefficients, after decryption."""
    g = gpu_small
    rng = np.random.default_rng(3)
    z = [rng.uniform(-1, 1, g.slots) for _ in range(3)]
    cts = [g.encrypt(g.encode(v, 4), 50 + k) for k, v in enumerate(z)]
    assert np.abs(g.decrypt(g.add_const(cts[0], -2.25)) - (z[0] - 2.25)).max() < 2.0 ** -20
    got = g.rescale(g.combine(cts, [0.5, -3.0, 1e-3], 7.125))
    assert np.abs(g.decrypt(got) - (0.5 * z[0] - 3.0 * z[1] + 1e-3 * z[2] + 7.125)).max() < 2.0 ** -20 and g.ct_meta(got)[0] == 3


def test_constants_that_are_refused(pkg, gpu_small, gpu_mid):
    g = gpu_small
    x, low, raw = _ct(g, _rand(g, 3, 2, 1)), _ct(g, _rand(g, 2, 2, 1)), _ct(g, _rand(g, 3, 2, 1), 2)
    for code, call in ((-1, lambda: g.add_const(x, float("nan"))), (-1, lambda: g.add_const(x, float("inf"))), (-9, lambda: g.add_const(x, 2.0 ** 21)), (-3, lambda: g.add_const(raw, 1.0)),
                       (-1, lambda: g.combine([x], [float("nan")])), (-9, lambda: g.combine([x], [-2.0 ** 21])), (-9, lambda: g.combine([x], [1.0], 2.0 ** 21)), (-2, lambda: g.combine([x, low], [1.0, 1.0])),
                       (-9, lambda: g.combine([], [])), (-9, lambda: g.combine([x] * 17, [1.0] * 17)), (-1, lambda: g.combine([_ct(gpu_mid, _rand(gpu_mid, 3, 2, 1))], [1.0]))):
        with pytest.raises(pkg.HBError) as e:
            call()
        assert e.value.code == code, e.value
    with pytest.raises(ValueError):
        g.combine([x], [1.0, 2.0])
    assert g._fn("combine")(g.ctx, (C.c_void_p * 1)(x.ptr.value), None, 1, C.c_double(0.0), C.byref(C.c_void_p())) == -1
    assert g._fn("add_const")(g.ctx, None, C.c_double(0.0), C.byref(C.c_void_p())) == -1


@pytest.mark.parametrize("members", [1, 3, 5])
@pytest.mark.parametrize("steps", [[0], [5], [0, 1, 2, 3], [-1, -2, -3, 0], [7, 7, 0], list(range(1, 17)) + [0]])
def test_sums_of_rotations_of_one_ciphertext(pkg, gpu_small, members, steps):
    g = gpu_small
    x = _ct(g, _rand(g, 4, members, 1))
    g.gen_rot_keys(steps)
    digits = g.decompose(x)
    if sum(s == 0 for s in steps) <= 16 and len(steps) <= 32:
        assert np.array_equal(g.ct_export(g.rotate_sum_hoisted(x, digits, steps)), g.ct_export(g.rotate_sum([x] * len(steps), steps)))
    with pytest.raises(pkg.HBError):   # digits of another ciphertext
        g.rotate_sum_hoisted(_ct(g, _rand(g, 3, members, 1)), digits, steps)
    with pytest.raises(pkg.HBError):
        g.rotate_sum_hoisted(x, digits, [])
    with pytest.raises(pkg.HBError):
        g.rotate_sum_hoisted(x, digits, [1] * 17)


def _device(handle, shape):
    import torch
    ptr = handle.lib._fn("ct_device_ptr")
    ptr.restype = C.c_void_p

    class View:
        __cuda_array_interface__ = {"shape": shape, "typestr": "<i8", "data": (ptr(handle.ptr), False), "version": 3, "strides": None}

    return torch.as_tensor(View(), device="cuda")


def test_more_members_than_a_grid_has_rows(pkg, gpu_small):
    """70000 token tiles of one column tile: past 65535 the sums take more of them a CTA, and calls that go member by member are refused."""
    import torch
    g, B, q = gpu_small, 70000, int(gpu_small.primes[0])
    x, m = g.ct_create(0, 2, B), g.ct_create(0, 2, B)
    for k, h in enumerate((x, m)):
        _device(h, (B, 2, 1, g.N)).random_(0, q, generator=torch.Generator(device="cuda").manual_seed(k))
    torch.cuda.synchronize()
    at, some = np.array([0, 1, 511, 512, g.N - 1]), [0, 1, 65534, 65535, 65536, B - 1]
    xo, mo = ({b: g.ct_export(g.batch_slice(h, b, 1))[0][..., at].astype(object) for b in some} for h in (x, m))

    def same(handle, want, polys):
        assert g.ct_meta(handle)[1:3] == (polys, B)
        for b in some:
            assert np.array_equal(g.ct_export(g.batch_slice(handle, b, 1))[0][..., at].astype(object), want(b) % q)

    same(g.norm_squares(x, 1, mean=m), lambda b: _pair(xo[b] - mo[b], xo[b] - mo[b]), 3)
    p = _rand(g, 0, 1, 5, polys=1)[0, 0]
    pt, po = _pt(g, p), p[..., at].astype(object)
    same(g.norm_affine(x, 1, gamma=[pt]), lambda b: np.stack([xo[b][0] * po, xo[b][1] * po]), 2)
    rows, rowsum, cols, colsum = g.norm_grad_sums(x, m, 1)
    same(rows, lambda b: _pair(xo[b], mo[b]), 3)
    same(rowsum, lambda b: xo[b], 2)
    want = (_device(x, (B, 2, 1, g.N))[:, 0, 0, at].cpu().numpy().astype(object).sum(0)) % q
    assert np.array_equal(g.ct_export(colsum)[0, 0, 0, at].astype(object), want)
    for call in (lambda: g.norm_scale(x, m, 1), lambda: g.norm_grad_input(x, m, x, m, 1), lambda: g.add_const(x, 1.0)):
        with pytest.raises(pkg.HBError) as e:
            call()
        assert e.value.code == -9
    del x, m, rows, rowsum, cols, colsum
    g._chk(g._fn("release_cached")(g.ctx))


def test_views_and_whole_calls_of_the_library_agree(gpu_small):
    """Runs of members without a copy as operands, and the residues of hb_tensor, hb_sub and hb_add."""
    g = gpu_small
    T, B, level = 3, 2, 4
    x, m, r = _ct(g, _rand(g, level, T * B + 3, 1)), _ct(g, _rand(g, level, B, 2)), _ct(g, _rand(g, level, B, 3))
    view = g._op("batch_view", x.ptr, C.c_int(2), C.c_int(T * B))
    acc = None
    for t in range(T):
        d = g.sub(g._op("batch_view", view.ptr, C.c_int(t * B), C.c_int(B)), m)
        assert np.array_equal(g.ct_export(g.tensor(d, r)), g.ct_export(g.norm_scale(view, r, T, mean=m))[t * B:(t + 1) * B])
        acc = g.tensor(d, d) if acc is None else g.add(acc, g.tensor(d, d))
    assert np.array_equal(g.ct_export(acc), g.ct_export(g.norm_squares(view, T, mean=m)))


def test_replayed_from_a_graph(gpu_small):
    g = gpu_small
    T, B, level = 4, 2, 3
    res = {k: _rand(g, level, n, s) for s, (k, n) in enumerate([("x", T * B), ("y", T * B), ("m", B), ("r", B), ("f", 1)])}
    h = {k: _ct(g, v) for k, v in res.items()}
    pts = [_pt(g, v[0]) for v in _rand(g, level, T, 9, polys=1)]

    def all_calls():
        return [g.norm_squares(h["x"], T, mean=h["m"], pad=3), g.norm_scale(h["x"], h["r"], T, mean=h["m"]), g.norm_affine(h["x"], T, gamma=pts, beta=pts),
                *g.norm_grad_sums(h["x"], h["y"], T), g.norm_grad_input(h["x"], h["m"], h["y"], h["r"], T), g.square_sum_many([h["x"], h["r"]]), *g.scale_many([h["x"], h["m"]], h["f"]),
                g.combine([h["x"], h["y"]], [0.5, -2.0])]

    want = [g.ct_export(o) for o in all_calls()]
    g.graph_begin()
    outs = all_calls()
    graph = g.graph_end()
    for k in h:   # other values while the graph does not run, then its own again
        g.ct_import(h[k], np.zeros_like(res[k]))
    g.graph_launch(graph)
    assert all(not g.ct_export(o).any() for o in outs[:2] + outs[3:])   # the affine part keeps its addend
    for k in h:
        g.ct_import(h[k], res[k])
    for _ in range(2):
        g.graph_launch(graph)
    for o, w in zip(outs, want):
        assert np.array_equal(g.ct_export(o), w)


def test_two_contexts_at_once(pkg, gpu_small):
    """Calls of two contexts from two threads, each on its own stream, while the other's are under way."""
    import threading
    other = pkg.open_gpu(pkg.make_params(log_n=12, max_level=8, dnum=3, num_special=3, hamming_weight=64))
    try:
        jobs, wrong = [], []
        for g, T, B in ((gpu_small, 5, 3), (other, 12, 4)):
            x, y, m, r = (_ct(g, _rand(g, 3, n, s)) for s, n in enumerate((T * B, T * B, B, B)))

            def calls(g=g, T=T, x=x, y=y, m=m, r=r):
                outs = [g.norm_squares(x, T, mean=m), g.norm_scale(x, r, T, mean=m), *g.norm_grad_sums(x, y, T), g.norm_grad_input(x, m, y, r, T), g.square_sum_many([x, y]), *g.scale_many([x, m], g.batch_slice(r, 0, 1))]
                return [g.ct_export(o) for o in outs]

            jobs.append((calls, calls()))

        def work(calls, want):
            for _ in range(20):
                if not all(np.array_equal(a, b) for a, b in zip(calls(), want)):
                    wrong.append(calls)

        threads = [threading.Thread(target=work, args=job) for job in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong
    finally:
        other.close()


def test_refusals(pkg, gpu_small, gpu_mid):
    g, level, T, B = gpu_small, 3, 2, 2
    x, m, f = _ct(g, _rand(g, level, T * B, 1)), _ct(g, _rand(g, level, B, 2)), _ct(g, _rand(g, level, 1, 3))
    low, three, raw = _ct(g, _rand(g, level - 1, B, 4)), _ct(g, _rand(g, level, B, 5, polys=3), 2), _ct(g, _rand(g, level, B, 6), 2)
    other = _ct(gpu_mid, _rand(gpu_mid, level, B, 7))
    p, plow = [_pt(g, _rand(g, level, 1, 8, polys=1)[0, 0])] * 2, [_pt(g, _rand(g, level - 1, 1, 8, polys=1)[0, 0])] * 2
    ARG, LEVEL, SHAPE = -1, -2, -3

    def refused(code, call, *a, **k):
        before = g.ct_export(x)
        with pytest.raises(pkg.HBError) as e:
            call(*a, **k)
        assert e.value.code == code, e.value
        assert np.array_equal(g.ct_export(x), before)

    for groups in (0, -1, 3, 5):
        refused(SHAPE, g.norm_squares, x, groups)
        refused(SHAPE, g.norm_scale, x, m, groups)
        refused(SHAPE, g.norm_grad_sums, x, x, groups)
        refused(SHAPE, g.norm_grad_input, x, m, x, m, groups)
    for groups in (3, 5):
        refused(SHAPE, g.norm_affine, x, groups, gamma=p[:1] * groups)
    refused(SHAPE, g._op, "norm_affine", x.ptr, None, None, C.c_int(0))
    for bad, code in ((low, LEVEL), (three, SHAPE), (raw, SHAPE), (other, ARG), (x, SHAPE), (f, SHAPE)):
        refused(code, g.norm_squares, x, T, mean=bad)
        if bad is not x:   # a factor per member
            refused(code, g.norm_scale, x, bad, T)
        refused(code, g.norm_scale, x, m, T, mean=bad)
        refused(code, g.norm_grad_input, x, bad, x, m, T)
        refused(code, g.norm_grad_input, x, m, x, bad, T)
        if bad is not x:
            refused(code, g.norm_grad_input, x, m, bad, m, T)
            refused(code, g.norm_grad_sums, x, bad, T)
            refused(code, g.norm_grad_sums, x, x, T, g=bad)
    refused(ARG, g.norm_squares, x, T, pad=1)
    refused(ARG, g.norm_squares, x, T, mean=m, pad=-1)
    refused(ARG, g.norm_squares, x, T, mean=m, pad=g.slots + 1)
    refused(ARG, g.norm_affine, x, T)
    refused(LEVEL, g.norm_affine, x, T, gamma=plow)
    refused(LEVEL, g.norm_affine, x, T, gamma=p, beta=plow)
    refused(ARG, g.square_sum_many, [])
    refused(ARG, g.scale_many, [], f)
    for bad, code in ((low, LEVEL), (three, SHAPE), (raw, SHAPE), (other, ARG)):
        refused(code, g.square_sum_many, [x, bad])
        refused(code, g.scale_many, [x, bad], f)
    refused(SHAPE, g.scale_many, [x], m)
    refused(LEVEL, g.scale_many, [x], _ct(g, _rand(g, level - 1, 1, 4)))
    with pytest.raises(ValueError):
        g.norm_affine(x, T, gamma=p[:1])
    with pytest.raises(ValueError):
        g.norm_squares(x, 2 ** 32 + 2)
    # nulls through the C entries
    out, null = C.c_void_p(), (C.c_void_p * 2)()
    for name, args in (("norm_squares", (None, None, 1, 0)), ("norm_scale", (x.ptr, None, None, 2)), ("norm_grad_input", (x.ptr, None, x.ptr, m.ptr, 2)), ("norm_affine", (x.ptr, null, None, 2)),
                       ("square_sum_many", (null, 2)), ("square_sum_many", (None, 2)), ("norm_grad_sums", (x.ptr, None, None, 2))):
        extra = [C.byref(out)] * (4 if name == "norm_grad_sums" else 1)
        assert g._fn(name)(g.ctx, *args, *extra) == ARG and not out.value
        assert g._fn(name)(g.ctx, *args, *[None] * len(extra)) == ARG
    assert g._fn("scale_many")(g.ctx, null, 2, f.ptr, null) == ARG
    assert g._fn("scale_many")(g.ctx, (C.c_void_p * 1)(x.ptr.value), 1, f.ptr, None) == ARG
