"""Products of a transformer block beyond one tile, decrypted, against products in 64 bits: query tiles against key tiles of another number, experts with
4-bit weights, encrypted vectors times a 4-bit matrix, and a run of them together.

Decrypted values may be off by 2^-14, the bound that every decrypted product of this repository is held to; sums over r tiles by r times that."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -14
D = 32  # the tile of the ring with 2^12 coefficients


@pytest.fixture(scope="module", params=[0, 1, 2])
def hemmer(request, pkg, gpu_mid):
    h = pkg.open_hemmer(gpu_mid)
    h.set_schedule(request.param)
    yield h
    h.close()


@pytest.fixture(scope="module")
def fast(pkg, gpu_mid):
    h = pkg.open_hemmer(gpu_mid)
    h.set_schedule(2)
    yield h
    h.close()


def _pairs(rng, count, scale=1.0):
    return [(rng.uniform(-scale, scale, (D, D)), rng.uniform(-scale, scale, (D, D))) for _ in range(count)]


def _encrypt(h, pairs, base):
    return h.encrypt2_many(pairs, [base + k for k in range(len(pairs))])


def _tiles(h, t):
    z = h.lib.decrypt_many([(t.ct, k) for k in range(h.lib.ct_meta(t.ct)[2])])[:, : 2 * D * D].real.reshape(-1, D, 2 * D)
    return z[:, :, :D], z[:, :, D:]


def _member(h, t, k):
    return type(t)(h.lib.batch_get(t.ct, k), *t.shape)


@pytest.mark.parametrize("heads,nq,nk", [(1, 1, 1), (2, 1, 3), (1, 3, 2), (2, 2, 2)])
def test_cross_scores(hemmer, heads, nq, nk):
    h, target = hemmer, 2
    rng = np.random.default_rng(heads + 10 * nq + 100 * nk)
    q, k = _pairs(rng, heads * nq), _pairs(rng, heads * nk)
    eq, ek = _encrypt(h, q, 100), _encrypt(h, k, 500)
    got = h.cross_scores(eq, ek, heads=heads, target_level=target)
    assert h.lib.ct_meta(got.ct)[:3] == (target, 2, heads * nq * nk)
    left, right = _tiles(h, got)
    for j, hd, i in np.ndindex(nk, heads, nq):
        (q0, q1), (k0, k1) = q[hd * nq + i], k[hd * nk + j]
        m = (j * heads + hd) * nq + i
        assert np.abs(left[m] - q0 @ k0.T).max() < TOL and np.abs(right[m] - q1 @ k1.T).max() < TOL
    # a pair does not depend on the others: the same bits alone
    i, j, hd = nq - 1, nk - 1, heads - 1
    alone = h.cross_scores(_member(h, eq, hd * nq + i), _member(h, ek, hd * nk + j), target_level=target)
    assert np.array_equal(h.lib.ct_export(alone.ct)[0], h.lib.ct_export(got.ct)[(j * heads + hd) * nq + i])


@pytest.mark.parametrize("heads,nq,nk,inner", [(1, 1, 1, 3), (2, 2, 1, 2), (1, 2, 3, 2)])
def test_cross_matmul_sums(hemmer, heads, nq, nk, inner):
    """Blocks of two matrices: the sum over the inner tiles."""
    h, target = hemmer, 2
    rng = np.random.default_rng(inner)
    a, b = _pairs(rng, inner * heads * nq), _pairs(rng, inner * heads * nk)
    left, right = _tiles(h, h.cross_matmul(_encrypt(h, a, 100), _encrypt(h, b, 500), heads=heads, inner=inner, target_level=target))
    for j, hd, i in np.ndindex(nk, heads, nq):
        m = (j * heads + hd) * nq + i
        for half, got in enumerate((left, right)):
            expected = sum(a[(r * heads + hd) * nq + i][half] @ b[(r * heads + hd) * nk + j][half] for r in range(inner))
            assert np.abs(got[m] - expected).max() < inner * TOL


def test_cross_matmul_of_thin_tiles(fast):
    """Heads narrower than the tile, as zero-padded columns; and the operands unchanged."""
    h, rng = fast, np.random.default_rng(3)
    pad = lambda m: np.pad(m, ((0, 0), (0, D - m.shape[1])))
    q, k = [(pad(a[:, :8]), pad(b[:, :8])) for a, b in _pairs(rng, 1)], [(pad(a[:, :8]), pad(b[:, :8])) for a, b in _pairs(rng, 2)]
    eq, ek = _encrypt(h, q, 1), _encrypt(h, k, 50)
    before = h.lib.ct_export(eq.ct), h.lib.ct_export(ek.ct)
    left, _ = _tiles(h, h.cross_scores(eq, ek, target_level=2))
    assert all(np.abs(left[j] - q[0][0] @ k[j][0].T).max() < TOL for j in range(2))
    assert np.array_equal(before[0], h.lib.ct_export(eq.ct)) and np.array_equal(before[1], h.lib.ct_export(ek.ct)) and ek.shape == (D, D, 2 * D)


def test_cross_refusals(pkg, fast):
    h, rng = fast, np.random.default_rng(4)
    a, b = _encrypt(h, _pairs(rng, 3), 1), _encrypt(h, _pairs(rng, 2), 50)
    for kw in (dict(heads=2), dict(heads=0), dict(inner=2), dict(inner=-1), dict(heads=3, inner=3), dict(target_level=6)):
        with pytest.raises(pkg.HBError) as e:
            h.cross_matmul(a, b, **kw)
        assert e.value.code == -1, kw
    with pytest.raises(pkg.HBError):
        h.cross_matmul(a, pkg.CtxtTensor(b.ct, D // 2, D, 2 * D))
    assert h.cross_matmul(a, b, target_level=2) is not None


def _matrix4(rng, rows, cols, group):
    """(codes, scales, the matrix they stand for): scales as a matrix of N(0, 0.05^2) has them"""
    w = rng.normal(0, 0.05, (rows, cols))
    groups = -(-rows // group)
    padded = np.zeros((groups * group, cols))
    padded[:rows] = w
    scales = (np.abs(padded).reshape(groups, group, cols).max(1) / 7).astype(np.float32)
    steps = np.clip(np.rint(w / np.repeat(scales.astype(np.float64), group, 0)[:rows]), -8, 7).astype(int)
    code = np.zeros((2 * -(-rows // 2), cols), dtype=np.uint8)
    code[:rows] = steps + 8
    return code[0::2] | (code[1::2] << 4), scales, steps * np.repeat(scales.astype(np.float64), group, 0)[:rows]


@pytest.mark.parametrize("rows,cols,group,vectors", [(1, 1, 1, 1), (4 * D, D, 32, 2), (300, 70, 48, 1), (257, 33, 64, 3)])
def test_vectors_times_4_bit_matrices(hemmer, rows, cols, group, vectors):
    h, rng = hemmer, np.random.default_rng(rows)
    codes, scales, w = _matrix4(rng, rows, cols, group)
    x = rng.uniform(-1, 1, (vectors, rows))
    ct = h.encrypt_vectors(x, 4, [900 + k for k in range(vectors * -(-rows // (4 * D)))])
    y = h.matvec_q4(ct, h.lib.qweight(codes, scales, rows, group))
    assert h.lib.ct_meta(y.ct)[0] == 3
    assert np.abs(h.decrypt_vectors(y, cols) - x @ w).max() < TOL


def test_matvec_refuses_other_batches(pkg, fast):
    h, rng = fast, np.random.default_rng(5)
    codes, scales, w = _matrix4(rng, 300, 10, 16)
    qw = h.lib.qweight(codes, scales, 300, 16)
    ct = h.encrypt_vectors(rng.uniform(-1, 1, (1, 100)), 3, [1])
    with pytest.raises(pkg.HBError):
        h.matvec_q4(ct, qw)


def test_grouped_refuses_null_arguments(fast):
    h = fast
    f, pre = h._fn("matmul_reuse_grouped"), h.lib.ct_create(2, 2, 2, 1)
    p = h.lib.encode(np.ones(4), 2)
    arr, sizes, out = (C.c_void_p * 1)(p.ptr.value), (C.c_int32 * 1)(2), C.c_void_p()
    args = lambda pre, sizes, arr, out: (h.h, pre, C.c_int(2), None, sizes, C.c_int(1), arr, C.c_int(1), C.c_int(1), C.c_int(2 * D), out)
    assert f(*args(pre.ptr, sizes, arr, None)) != 0 and f(*args(None, sizes, arr, C.byref(out))) != 0
    assert f(*args(pre.ptr, None, arr, C.byref(out))) != 0 and f(*args(pre.ptr, sizes, None, C.byref(out))) != 0
    assert out.value is None and f(*args(pre.ptr, sizes, arr, C.byref(out))) == 0
    type(p)(h.lib, out, "ct")


def test_a_block_of_them(fast):
    """An encrypted block with more than one tile: three sequences at two of three experts with 4-bit weights; the scores of one tile of queries against two of
    keys and their product with the values; the last vector through a 4-bit head.  Between the products the values come back to the client, as in the layer
    workload, whose products all start from freshly encrypted operands."""
    h, target = fast, 2
    lib, rng = h.lib, np.random.default_rng(6)
    rows, cols, inputs = 4 * D, 2 * D, 3
    # experts: the operands of 128 x 64 matrices from their codes
    experts, weights = [], []
    for e in range(3):
        codes, scales, w = _matrix4(rng, rows, cols, 32)
        experts.append(w)
        weights.append(h.encode_diagonal_to_row4_q4(lib.qweight(codes, scales, rows, 32), rows, cols, level=target + 1))
    x = rng.uniform(-1, 1, (inputs, D, rows))
    tiles = lambda m, c: m[:, c * D:(c + 1) * D]
    packed = h.complex_packing(_encrypt(h, [(tiles(x[i], 0), tiles(x[i], 1)) for i in range(inputs)], 10), _encrypt(h, [(tiles(x[i], 2), tiles(x[i], 3)) for i in range(inputs)], 60))
    pre = h.matmul_pre(packed, target)
    sizes, order = [2, 0, 3], [0, 2, 1, 0, 2]
    y = h.matmul_reuse_experts(pre, inputs, sizes, [weights[0], None, weights[2]], order=order)
    left, right = _tiles(h, y)
    at = [e for e, n in enumerate(sizes) for _ in range(n)]
    expected = [x[i] @ experts[e] for i, e in zip(order, at)]
    out = 2 * (left + right)
    for p, t in np.ndindex(len(order), 2):
        assert np.abs(out[2 * p + t] - tiles(expected[p], t)).max() < TOL
    # the same weights encoded from doubles give the same bits
    one = experts[2]
    same = h.matmul_reuse(lib_member(h, pre, inputs, 1), h.encode_diagonal_to_row4(*[one[i * D:(i + 1) * D, :D] for i in range(4)], level=target + 1))
    assert np.array_equal(lib.ct_export(same.ct)[0], lib.ct_export(y.ct)[2 * 2])
    # attention of the first sequence's tile to the other two
    scale = 0.2
    q, k, v = [scale * out[0]], [scale * out[4], scale * out[6]], [out[5], out[7]]
    eq, ek, ev = (_encrypt(h, [(t, t) for t in ts], base) for ts, base in ((q, 200), (k, 300), (v, 400)))
    s, _ = _tiles(h, h.cross_scores(eq, ek, target_level=target))
    assert all(np.abs(s[j] - q[0] @ k[j].T).max() < TOL for j in range(2))
    p = np.exp(np.concatenate([s[0], s[1]], axis=1))
    p /= p.sum(1, keepdims=True)
    probs = _encrypt(h, [(p[:, :D], p[:, :D]), (p[:, D:], p[:, D:])], 500)
    z, _ = _tiles(h, h.cross_matmul(probs, ev, inner=2, target_level=target))
    assert np.abs(z[0] - p @ np.concatenate(v)).max() < 2 * TOL
    # the last token through the head
    codes, scales, head = _matrix4(rng, D, 10, 16)
    last = h.matvec_q4(h.encrypt_vectors(z[0][-1:], 3, [600]), lib.qweight(codes, scales, D, 16))
    assert np.abs(h.decrypt_vectors(last, 10) - z[0][-1:] @ head).max() < TOL


def lib_member(h, pre, inputs, i):
    """The shifted copies of input i out of those of `inputs`."""
    copies = h.lib.ct_meta(pre)[2] // inputs
    return h.lib.batch_concat([h.lib.batch_get(pre, k * inputs + i) for k in range(copies)])
