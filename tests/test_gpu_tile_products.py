"""hb_tensor_acc_cross and hb_matmul_acc_grouped against sums of products of Python's own integers, member by member, and against the calls that
do the same pair by pair or input by input.  All results are whole numbers: equal or wrong."""
import ctypes as C

import numpy as np
import pytest

from conftest import rand_ct_residues

pytestmark = pytest.mark.gpu

U64 = np.uint64


def _ct(g, res, scale_pow=1):
    ct = g.ct_create(res.shape[2] - 1, res.shape[1], res.shape[0], scale_pow)
    g.ct_import(ct, res)
    return ct


def _pt(g, res):
    """A plaintext with given residues: any plaintext of the level, its one-polynomial words replaced through the device pointer's owner."""
    import torch
    pt = g.encode(np.zeros(1), res.shape[0] - 1)
    ptr = g._fn("pt_device_ptr")
    ptr.restype = C.c_void_p

    class View:
        __cuda_array_interface__ = {"shape": res.shape, "typestr": "<i8", "data": (ptr(pt.ptr), False), "version": 3, "strides": None}

    torch.as_tensor(View(), device="cuda").copy_(torch.from_numpy(res.astype(np.int64)))
    torch.cuda.synchronize()
    return pt


def _rand(g, level, batch, seed, polys=2, edge=False):
    res = rand_ct_residues(g, level, polys, batch, seed)
    if edge:  # the largest residues there are: every partial sum as large as it gets
        res[:] = np.array([int(q) - 1 for q in g.primes[: level + 1]], dtype=U64)[None, None, :, None]
    return res


def _points(g, rng, n=40):
    """Coefficients to check: the first and last, and a random choice (every coefficient goes through the same arithmetic on its own thread)."""
    return np.unique(np.concatenate([[0, 1, 31, 32, 255, 256, g.N - 1], rng.integers(0, g.N, n)]))


def _cross_expected(a, b, groups, heads, primes, at):
    nq, nk, n = a.shape[0] // (groups * heads), b.shape[0] // (groups * heads), a.shape[2]
    a = a[..., at].astype(object).reshape(groups, heads, nq, 2, n, at.size)
    b = b[..., at].astype(object).reshape(groups, heads, nk, 2, n, at.size)
    q = np.array([int(p) for p in primes[:n]], dtype=object)[:, None]
    out = np.empty((nk, heads, nq, 3, n, at.size), dtype=object)
    for j, h, i in np.ndindex(nk, heads, nq):
        x, y = a[:, h, i], b[:, h, j]
        out[j, h, i, 0] = (x[:, 0] * y[:, 0]).sum(0) % q
        out[j, h, i, 1] = (x[:, 0] * y[:, 1] + x[:, 1] * y[:, 0]).sum(0) % q
        out[j, h, i, 2] = (x[:, 1] * y[:, 1]).sum(0) % q
    return out.reshape(-1, 3, n, at.size)


def _same(got, expected, at):
    assert np.array_equal(got[..., at].astype(object), expected)


SHAPES = [  # groups, heads, query tiles, key tiles
    (1, 1, 1, 1), (1, 2, 1, 2), (3, 1, 2, 1), (2, 1, 2, 2), (5, 2, 3, 3), (2, 1, 1, 7), (4, 3, 5, 1), (7, 1, 4, 3), (33, 1, 1, 1), (65, 1, 2, 3), (2, 1, 8, 9),
]


@pytest.mark.parametrize("groups,heads,nq,nk", SHAPES)
def test_cross_small_ring(gpu_small, groups, heads, nq, nk):
    g = gpu_small
    rng = np.random.default_rng(groups * 1000 + nq * 10 + nk)
    a, b = _rand(g, 3, groups * heads * nq, 1), _rand(g, 3, groups * heads * nk, 2)
    at = _points(g, rng, 12)
    got = g.ct_export(g.tensor_acc_cross(_ct(g, a), _ct(g, b), groups, heads=heads))
    _same(got, _cross_expected(a, b, groups, heads, g.primes, at), at)


@pytest.mark.parametrize("groups", [1, 2, 31, 32, 33, 64, 97])
def test_cross_largest_residues(gpu_mid, groups):
    """Every residue q - 1: sums as large as they get, on both sides of the counts after which they are reduced."""
    g = gpu_mid
    a, b = _rand(g, 8, groups * 2, 1, edge=True), _rand(g, 8, groups * 2, 2, edge=True)
    at = np.array([0, 5, g.N - 1])
    got = g.ct_export(g.tensor_acc_cross(_ct(g, a), _ct(g, b), groups))
    _same(got, _cross_expected(a, b, groups, 1, g.primes, at), at)


@pytest.mark.parametrize("level,groups,heads,nq,nk", [(0, 4, 1, 2, 2), (5, 8, 2, 1, 4), (5, 3, 1, 4, 1), (12, 2, 1, 3, 2), (2, 9, 1, 5, 5)])
def test_cross_full_ring(gpu_full, level, groups, heads, nq, nk):
    g = gpu_full
    rng = np.random.default_rng(level)
    a, b = _rand(g, level, groups * heads * nq, 3), _rand(g, level, groups * heads * nk, 4)
    at = _points(g, rng)
    ca, cb = _ct(g, a), _ct(g, b)
    got = g.ct_export(g.tensor_acc_cross(ca, cb, groups, heads=heads))
    _same(got, _cross_expected(a, b, groups, heads, g.primes, at), at)
    # every coefficient: the pairs one by one
    take = lambda ct, of, i: g.batch_concat([g.batch_get(ct, (gr * heads + h) * of + i) for gr in range(groups) for h in range(heads)])
    for i, j in {(0, 0), (nq - 1, nk - 1), (nq // 2, nk - 1)}:
        out = C.c_void_p()
        x, y = take(ca, nq, i), take(cb, nk, j)
        g._chk(g.dll.hb_tensor_acc_groups(g.ctx, x.ptr, y.ptr, C.c_int(groups), C.byref(out)))
        single = g.ct_export(type(x)(g, out, "ct"))
        for h in range(heads):
            assert np.array_equal(got[(j * heads + h) * nq + i], single[h])


OTHER_PRIMES = [dict(log_n=10, max_level=4, dnum=3, q_bits=43), dict(log_n=10, max_level=4, dnum=3, q_bits=44), dict(log_n=10, max_level=4, dnum=3, q_bits=46, p_bits=58),
                dict(log_n=11, max_level=4, dnum=3, q_bits=59), dict(log_n=16, max_level=3, dnum=3, q_bits=44), dict(log_n=16, max_level=3, dnum=3, q0_bits=58, q_bits=50, p_bits=58)]


@pytest.mark.parametrize("prm", OTHER_PRIMES)
def test_other_primes(pkg, prm):
    """Primes of 43 and 44 bits, whose sums have less room, and longer ones; the largest residues and uniform ones."""
    g = pkg.open_gpu(pkg.make_params(num_special=3, hamming_weight=32, **prm))
    try:
        rng = np.random.default_rng(1)
        at = np.unique(np.concatenate([[0, g.N - 1], rng.integers(0, g.N, 10)]))
        for edge in (False, True):
            for groups, nq, nk in ((1, 1, 1), (3, 2, 1), (9, 4, 3), (17, 1, 4), (34, 2, 2)):
                a, b = _rand(g, 3, groups * nq, 3, edge=edge), _rand(g, 3, groups * nk, 4, edge=edge)
                _same(g.ct_export(g.tensor_acc_cross(_ct(g, a), _ct(g, b), groups)), _cross_expected(a, b, groups, 1, g.primes, at), at)
            for copies, bcount, sizes, tiles in ((9, 1, [1], 8), (17, 1, [3, 1], 4), (9, 2, [2], 6)):
                pre, pts = _rand(g, 3, copies * 3 * bcount, 5, edge=edge), _weights(g, 3, len(sizes), tiles, bcount, 6)
                if edge:
                    pts[:] = np.array([int(q) - 1 for q in g.primes[:4]], dtype=U64)[None, None, None, :, None]
                order = list(range(sum(sizes)))
                order = [i % 3 for i in order]
                got = g.ct_export(g.matmul_acc_grouped(_ct(g, pre), 3, sizes, _handles(g, pts, sizes), 2, order=order))
                _same(got, _grouped_expected(g, pre, pts, copies, 3, sizes, order, 2, at), at)
    finally:
        g.close()


def test_cross_accumulates(gpu_small):
    """*acc += sum: in two halves the same as at once; the accumulator's handle stays the caller's."""
    g = gpu_small
    a, b = _rand(g, 4, 2 * 4 * 3, 5), _rand(g, 4, 2 * 4 * 2, 6)
    whole = g.ct_export(g.tensor_acc_cross(_ct(g, a), _ct(g, b), 4, heads=2))
    acc = g.tensor_acc_cross(_ct(g, a[:12]), _ct(g, b[:8]), 2, heads=2)
    assert g.tensor_acc_cross(_ct(g, a[12:]), _ct(g, b[8:]), 2, heads=2, acc=acc) is acc
    assert np.array_equal(g.ct_export(acc), whole)


def test_cross_of_views_and_of_one_ciphertext_twice(gpu_small):
    g = gpu_small
    x = _rand(g, 2, 10, 7)
    ct, at = _ct(g, x), np.arange(0, g.N, 37)
    v = C.c_void_p()
    g._chk(g.dll.hb_batch_view(g.ctx, ct.ptr, C.c_int(1), C.c_int(6), C.byref(v)))
    view = type(ct)(g, v, "ct")
    _same(g.ct_export(g.tensor_acc_cross(view, view, 2)), _cross_expected(x[1:7], x[1:7], 2, 1, g.primes, at), at)
    assert np.array_equal(g.ct_export(ct), x)


def test_cross_refusals(pkg, gpu_small, gpu_mid):
    g = gpu_small
    a, b = _ct(g, _rand(g, 2, 6, 1)), _ct(g, _rand(g, 2, 4, 2))
    cases = [
        (a, b, dict(groups=4), -3), (a, b, dict(groups=0), -3), (a, b, dict(groups=-2), -3), (a, b, dict(groups=2, heads=0), -3), (a, b, dict(groups=2, heads=2), -3),
        (a, _ct(g, _rand(g, 3, 4, 2)), dict(groups=2), -2), (a, g.ct_create(2, 3, 4, 1), dict(groups=2), -3), (g.ct_create(2, 2, 6, 2), b, dict(groups=2), -3),
        (a, b, dict(groups=2, acc=g.ct_create(2, 3, 5, 2)), -3), (a, b, dict(groups=2, acc=g.ct_create(2, 2, 6, 2)), -3), (a, b, dict(groups=2, acc=g.ct_create(1, 3, 6, 2)), -3),
        (a, gpu_mid.ct_create(2, 2, 4, 1), dict(groups=2), -1), (a, b, dict(groups=65536, heads=65536), -3),
    ]
    for x, y, kw, code in cases:
        with pytest.raises(pkg.HBError) as e:
            g.tensor_acc_cross(x, y, **kw)
        assert e.value.code == code, (kw, e.value)
    out = C.c_void_p()
    assert g.dll.hb_tensor_acc_cross(g.ctx, None, b.ptr, C.c_int(1), C.c_int(1), C.byref(out)) == -1
    assert g.dll.hb_tensor_acc_cross(g.ctx, a.ptr, None, C.c_int(1), C.c_int(1), C.byref(out)) == -1
    assert g.dll.hb_tensor_acc_cross(g.ctx, a.ptr, b.ptr, C.c_int(1), C.c_int(1), None) == -1
    assert g.tensor_acc_cross(a, b, 2) is not None  # the context goes on


# ---- products grouped by expert ----------------------------------------------------------------------------------------
def _turned(g, steps, at):
    """Where the coefficients `at` of a rotated plaintext come from: the transform's slot i is the value at psi^(2 bitrev(i) + 1)."""
    logn = g.N.bit_length() - 1
    rev = np.array([int(format(i, f"0{logn}b")[::-1], 2) for i in range(g.N)])
    gal = pow(5, steps % g.slots, 2 * g.N)
    return rev[(gal * (2 * rev[at] + 1) % (2 * g.N)) >> 1]


def _grouped_expected(g, pre, pts, copies, inputs, sizes, order, row_step, at):
    n, (experts, tiles, bcount) = pre.shape[2], pts.shape[:3]
    pre = pre.astype(object).reshape(copies, inputs, bcount, 2, n, -1)
    q = np.array([int(p) for p in g.primes[:n]], dtype=object)[:, None]
    expert = [e for e, size in enumerate(sizes) for _ in range(size)]
    turned = [_turned(g, k * row_step, at) for k in range(copies)]
    out = np.empty((len(expert), tiles, 2, n, at.size), dtype=object)
    for p, e in enumerate(expert):
        i = p if order is None else order[p]
        for t in range(tiles):
            acc = 0
            for k in range(copies):
                for b in range(bcount):
                    acc = acc + pre[k, i, b][..., at] * pts[e, t, b][:, turned[k]].astype(object)
            out[p, t] = acc % q
    return out.reshape(-1, 2, n, at.size)


def _handles(g, pts, sizes):
    return [[[_pt(g, pts[e, t, b]) for b in range(pts.shape[2])] for t in range(pts.shape[1])] if sizes[e] else None for e in range(pts.shape[0])]


def _weights(g, level, experts, tiles, bcount, seed):
    return rand_ct_residues(g, level, 1, experts * tiles * bcount, seed).reshape(experts, tiles, bcount, level + 1, g.N)


GROUPED = [  # copies, inputs, bcount, sizes, order, tiles
    (1, 1, 1, [1], None, 1),
    (4, 3, 1, [1, 1, 1], None, 1),
    (2, 3, 2, [0, 3, 0], None, 2),
    (3, 2, 1, [2, 0, 1, 1], [1, 0, 1, 1], 3),          # an input at several experts, and twice in a row
    (5, 4, 2, [4, 3, 0, 2], [0, 1, 2, 3, 3, 1, 0, 2, 2], 5),
    (2, 1, 1, [5], [0, 0, 0, 0, 0], 4),
    (16, 2, 3, [1, 2], [1, 0, 1], 6),
    (3, 2, 16, [1, 1], None, 2),                       # the most K-groups
    (2, 5, 1, [0, 0, 0, 0, 1], [4], 7),
    (6, 2, 1, [1, 1], None, 8), (6, 2, 1, [1, 1], None, 5), (7, 3, 2, [3], None, 6), (5, 3, 1, [6, 1, 3], [0, 1, 2, 0, 1, 2, 2, 1, 1, 0], 9), (3, 4, 1, [4], None, 12),
]


@pytest.mark.parametrize("copies,inputs,bcount,sizes,order,tiles", GROUPED)
def test_grouped_small_ring(gpu_small, copies, inputs, bcount, sizes, order, tiles):
    g = gpu_small
    rng = np.random.default_rng(copies + 10 * inputs)
    pre, pts = _rand(g, 2, copies * inputs * bcount, 1), _weights(g, 2, len(sizes), tiles, bcount, 2)
    at = _points(g, rng, 8)
    got = g.ct_export(g.matmul_acc_grouped(_ct(g, pre), inputs, sizes, _handles(g, pts, sizes), 32, order=order))
    _same(got, _grouped_expected(g, pre, pts, copies, inputs, sizes, order, 32, at), at)


@pytest.mark.parametrize("positions,experts,tiles,bcount", [(300, 3, 1, 1), (70, 70, 1, 1), (9, 2, 25, 16), (2, 2, 390, 1), (1, 1, 25, 16)])
def test_grouped_beyond_one_launch(gpu_small, positions, experts, tiles, bcount):
    """More positions, experts or weights than one launch lists."""
    g = gpu_small
    inputs, rng = 3, np.random.default_rng(positions)
    sizes = np.bincount(rng.integers(0, experts, positions) if experts < positions else np.arange(positions), minlength=experts).tolist()
    order = rng.integers(0, inputs, positions).tolist()
    pre, pts = _rand(g, 0, 2 * inputs * bcount, 3), _weights(g, 0, experts, tiles, bcount, 4)
    at = np.array([0, 77, g.N - 1])
    got = g.ct_export(g.matmul_acc_grouped(_ct(g, pre), inputs, sizes, _handles(g, pts, sizes), 8, order=order))
    _same(got, _grouped_expected(g, pre, pts, 2, inputs, sizes, order, 8, at), at)


@pytest.mark.parametrize("copies,bcount", [(8, 1), (9, 1), (127, 1), (128, 1), (129, 1), (65, 2), (17, 16)])
def test_grouped_largest_residues(gpu_small, copies, bcount):
    """Every word q - 1, on both sides of the counts after which sums are reduced."""
    g = gpu_small
    pre = _rand(g, 2, copies * 2 * bcount, 1, edge=True)
    pts = np.broadcast_to(pre[0, 0], (2, 3, bcount, 3, g.N)).copy()
    at = np.array([0, 9, g.N - 1])
    sizes = [2, 1]
    got = g.ct_export(g.matmul_acc_grouped(_ct(g, pre), 2, sizes, _handles(g, pts, sizes), 4, order=[0, 1, 1]))
    _same(got, _grouped_expected(g, pre, pts, copies, 2, sizes, [0, 1, 1], 4, at), at)


@pytest.mark.parametrize("level,copies,inputs,bcount,sizes,tiles", [(5, 6, 3, 1, [2, 0, 1], 3), (1, 128, 2, 2, [1, 1], 2), (12, 2, 2, 1, [2], 4), (0, 5, 5, 1, [3, 2], 1)])
def test_grouped_full_ring(gpu_full, level, copies, inputs, bcount, sizes, tiles):
    g = gpu_full
    rng = np.random.default_rng(level)
    pre, pts = _rand(g, level, copies * inputs * bcount, 5), _weights(g, level, len(sizes), tiles, bcount, 6)
    at, hs, ct = _points(g, rng, 20), _handles(g, pts, sizes), _ct(g, pre)
    got = g.ct_export(g.matmul_acc_grouped(ct, inputs, sizes, hs, 256))
    _same(got, _grouped_expected(g, pre, pts, copies, inputs, sizes, None, 256, at), at)
    # every coefficient: input by input
    p = 0
    for e, size in enumerate(sizes):
        for _ in range(size):
            arr = (C.c_void_p * bcount)(*[h.ptr.value for h in hs[e][tiles - 1]])
            out = C.c_void_p()
            g._chk(g.dll.hb_matmul_acc_multi(g.ctx, ct.ptr, C.c_int(inputs * bcount), C.c_int(p * bcount), arr, C.c_int(bcount), C.c_int64(256), C.byref(out)))
            assert np.array_equal(g.ct_export(type(ct)(g, out, "ct"))[0], got[p * tiles + tiles - 1])
            p += 1


def test_grouped_refusals(pkg, gpu_small, gpu_mid):
    g = gpu_small
    pre = _ct(g, _rand(g, 2, 12, 1))
    w = lambda level=2: [[g.encode(np.ones(4), level)] for _ in range(2)]
    one = [w(), w()]
    bad = [
        (dict(inputs=5, sizes=[1, 1], pts=one), -3), (dict(inputs=0, sizes=[1, 1], pts=one), -3), (dict(inputs=3, sizes=[4, 1], pts=one), -3),
        (dict(inputs=3, sizes=[1, -1], pts=one), -3), (dict(inputs=3, sizes=[1, 1], pts=one, order=[0, 3]), -1), (dict(inputs=3, sizes=[1, 1], pts=one, order=[-1, 0]), -1),
        (dict(inputs=3, sizes=[1, 1], pts=[w(), w(3)]), -2), (dict(inputs=4, sizes=[1], pts=[[[gpu_mid.encode(np.ones(4), 2)]]]), -1),
    ]
    for kw, code in bad:
        kw = dict(kw)
        with pytest.raises(pkg.HBError) as e:
            if min(kw["sizes"]) < 0:  # the wrapper sums the sizes: straight to the entry point
                arr = (C.c_void_p * 4)(*[p.ptr.value for rows in one for row in rows for p in row])
                out = C.c_void_p()
                g._chk(g.dll.hb_matmul_acc_grouped(g.ctx, pre.ptr, C.c_int(3), None, (C.c_int32 * 2)(*kw["sizes"]), C.c_int(2), arr, C.c_int(1), C.c_int(2), C.c_int64(8), C.byref(out)))
            g.matmul_acc_grouped(pre, row_step=8, **kw)
        assert e.value.code == code, (kw, e.value)
    for kw in (dict(sizes=[0, 0], pts=[None, None]), dict(sizes=[1], pts=one), dict(sizes=[1, 1], pts=[w(), w() + w()]), dict(sizes=[1, 1], pts=one, order=[0])):
        with pytest.raises(ValueError):
            g.matmul_acc_grouped(pre, 3, row_step=8, **kw)
    out, arr = C.c_void_p(), (C.c_void_p * 2)()
    f = g.dll.hb_matmul_acc_grouped
    size = lambda *v: (C.c_int32 * len(v))(*v)
    tail = (C.c_int(1), C.c_int(2), C.c_int64(8), C.byref(out))
    assert f(g.ctx, pre.ptr, C.c_int(3), None, size(1), C.c_int(1), arr, *tail) == -1         # null plaintexts of an expert with inputs
    assert f(g.ctx, pre.ptr, C.c_int(3), None, size(0), C.c_int(1), arr, *tail) == -3         # nobody has an input
    assert f(g.ctx, pre.ptr, C.c_int(3), None, None, C.c_int(1), arr, *tail) == -1
    assert f(g.ctx, None, C.c_int(3), None, size(1), C.c_int(1), arr, *tail) == -1
    assert f(g.ctx, pre.ptr, C.c_int(3), None, size(1), C.c_int(1), arr, C.c_int(17), C.c_int(1), C.c_int64(8), C.byref(out)) == -3
    raw = g.ct_create(2, 2, 12, 2)
    with pytest.raises(pkg.HBError) as e:
        g.matmul_acc_grouped(raw, 3, [1, 1], one, 8)
    assert e.value.code == -3


def test_recorded_products(gpu_small):
    """Both products recorded and replayed on changed operands; two graphs whose temporaries are the same idle buffers, replayed in turn."""
    g = gpu_small
    a, b = _rand(g, 2, 6, 1), _rand(g, 2, 4, 2)
    ca, cb = _ct(g, a), _ct(g, b)
    pts = _weights(g, 2, 2, 2, 1, 3)
    hs = _handles(g, pts, [1, 2])
    run = lambda: (g.tensor_acc_cross(ca, cb, 2), g.matmul_acc_grouped(ca, 3, [1, 2], hs, 32, order=[2, 0, 2]))
    run()
    graphs = []
    for _ in range(2):
        g.graph_begin()
        out = run()
        graphs.append((g.graph_end(), out))
    at = np.arange(0, g.N, 29)
    for seed in (11, 12):
        a, b = _rand(g, 2, 6, seed), _rand(g, 2, 4, seed + 50)
        g.ct_import(ca, a); g.ct_import(cb, b)
        for graph, _ in graphs:
            g.graph_launch(graph)
        g.sync()
        for _, (x, y) in graphs:
            _same(g.ct_export(x), _cross_expected(a, b, 2, 1, g.primes, at), at)
            _same(g.ct_export(y), _grouped_expected(g, a, pts, 2, 3, [1, 2], [2, 0, 2], 32, at), at)
