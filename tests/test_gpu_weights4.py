"""4-bit weights with group scales: the operands made on the device against hb_encode of the same values, bit for bit; products against sums of those;
decrypted matrix-vector products against a product in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from conftest import rand_ct_residues

pytestmark = pytest.mark.gpu


def _matrix(rows, cols, group, seed):
    """(codes as bytes, scales, the matrix they stand for); all sixteen codes, scales from tiny to large, a zero one and a negative one among them"""
    rng = np.random.default_rng(seed)
    code = rng.integers(0, 16, (rows, cols))
    scales = (rng.uniform(0.5, 1.5, (-(-rows // group), cols)) * 0.01).astype(np.float32)
    scales[0, 0] = 0.0
    scales[-1, -1] = -0.02
    scales[0, cols // 2] = np.float32(1e-42)  # below the normal range
    w = (code - 8).astype(np.float64) * np.repeat(scales.astype(np.float64), group, axis=0)[:rows]
    padded = np.zeros((2 * -(-rows // 2), cols), dtype=np.uint8)
    padded[:rows] = code
    return padded[0::2] | (padded[1::2] << 4), scales, w


def _slots(w, d, b, j, diagonal, slots):
    """Slot values of block (column tile j, K-group b)"""
    t = np.zeros((4 * d, d))
    part = w[4 * d * b:4 * d * (b + 1), d * j:d * (j + 1)]
    t[: part.shape[0], : part.shape[1]] = part
    w1, w2, w3, w4 = t.reshape(4, d, d)
    left, right = 0.5 * (w1 - 1j * w3), 0.5 * (w2 - 1j * w4)
    if diagonal:
        for c in range(d):
            left[:, c], right[:, c] = np.roll(left[:, c], -c), np.roll(right[:, c], -c)
    z = np.zeros(slots, dtype=np.complex128)
    z[: 2 * d * d] = np.concatenate([left, right], axis=1).reshape(-1)
    return z


def _tile(g):
    return 1 << ((g.N.bit_length() - 3) // 2)


MATRICES = [(1, 1, 1), (2, 3, 1), (7, 5, 3), (64, 16, 64), (65, 17, 16), (100, 33, 48), (129, 40, 1000), (3, 70, 2)]


@pytest.mark.parametrize("rows,cols,group", MATRICES)
@pytest.mark.parametrize("diagonal", [False, True])
def test_operands_small_ring(gpu_small, rows, cols, group, diagonal):
    g, d = gpu_small, _tile(gpu_small)
    codes, scales, w = _matrix(rows, cols, group, rows)
    qw = g.qweight(codes, scales, rows, group)
    kb, nb = -(-rows // (4 * d)), -(-cols // d)
    for level in (0, 3, 8):
        got = g.encode_q4(qw, d, 0, kb * nb, level, diagonal=diagonal)
        for j in range(nb):
            for b in range(kb):
                p = got[j * kb + b]
                assert g.pt_meta(p) == (level, 1)
                assert np.array_equal(g.pt_export(p), g.pt_export(g.encode(_slots(w, d, b, j, diagonal, g.slots), level))), (level, j, b)


@pytest.mark.parametrize("rows,cols,group,level", [(768, 256, 128, 5), (513, 129, 48, 12), (1, 1, 1, 0), (100, 300, 7, 2)])
@pytest.mark.parametrize("diagonal", [False, True])
def test_operands_full_ring(gpu_full, rows, cols, group, level, diagonal):
    g, d = gpu_full, 128
    codes, scales, w = _matrix(rows, cols, group, rows)
    qw = g.qweight(codes, scales, rows, group)
    kb, nb = -(-rows // (4 * d)), -(-cols // d)
    got = g.encode_q4(qw, d, 0, kb * nb, level, diagonal=diagonal)
    for j in range(nb):
        for b in range(kb):
            assert np.array_equal(g.pt_export(got[j * kb + b]), g.pt_export(g.encode(_slots(w, d, b, j, diagonal, g.slots), level))), (j, b)


@pytest.mark.parametrize("tile", [1, 3, 8, 15])
def test_operands_of_other_tiles(gpu_small, tile):
    """Any side of which two tiles fit the slots; more blocks than are encoded at a time; runs that begin inside."""
    g = gpu_small
    codes, scales, w = _matrix(37, 29, 5, tile)
    qw = g.qweight(codes, scales, 37, 5)
    kb, nb = -(-37 // (4 * tile)), -(-29 // tile)
    count = min(kb * nb, 75)
    got = g.encode_q4(qw, tile, 0, count, 1)
    part = g.encode_q4(qw, tile, count // 2, 1, 1)[0]
    assert np.array_equal(g.pt_export(part), g.pt_export(got[count // 2]))
    for k in sorted({0, 1, count // 3, count - 1} & set(range(count))):
        assert np.array_equal(g.pt_export(got[k]), g.pt_export(g.encode(_slots(w, tile, k % kb, k // kb, True, g.slots), 1))), k


@pytest.mark.parametrize("ring", ["small", "full"])
@pytest.mark.parametrize("bits", [0, 6, 12, 16, 40, 100])
def test_operands_of_large_scales(request, ring, bits):
    """Coefficients on both sides of the magnitudes after which they are reduced another way (2^44, 2^50), and past 63 bits, where they are what hb_encode makes of them."""
    g = request.getfixturevalue("gpu_" + ring)
    d = _tile(g)
    codes, scales, _ = _matrix(4 * d + 5, d + 3, 16, bits)
    scales = (scales.astype(np.float64) * 2.0**bits).astype(np.float32)
    scales[0, 1] = np.float32(2.0**bits * 3)  # a few coefficients' worth above the others
    code = np.empty((2 * codes.shape[0], codes.shape[1]))
    code[0::2], code[1::2] = codes & 15, codes >> 4
    w = (code[: 4 * d + 5] - 8) * np.repeat(scales.astype(np.float64), 16, axis=0)[: 4 * d + 5]
    qw = g.qweight(codes, scales, 4 * d + 5, 16)
    got = g.encode_q4(qw, d, 0, 4, 2)
    for j, b in np.ndindex(2, 2):
        assert np.array_equal(g.pt_export(got[j * 2 + b]), g.pt_export(g.encode(_slots(w, d, b, j, True, g.slots), 2))), (j, b)


def _operand_sums(g, x, operands, kb, nb, at):
    """sum_b x[v][b] (.) p[j][b] in Python's integers"""
    n = x.shape[2]
    x = x[..., at].astype(object).reshape(-1, kb, 2, n, at.size)
    q = np.array([int(p) for p in g.primes[:n]], dtype=object)[:, None]
    p = [g.pt_export(h)[:, at].astype(object) for h in operands]
    out = np.empty((x.shape[0], nb, 2, n, at.size), dtype=object)
    for v, j in np.ndindex(x.shape[0], nb):
        out[v, j] = sum(x[v, b] * p[j * kb + b][None] for b in range(kb)) % q
    return out.reshape(-1, 2, n, at.size)


VECTORS = [(1, 1, 1, 1, 0), (7, 5, 3, 2, 1), (65, 17, 16, 1, 3), (200, 40, 48, 3, 2), (64 * 9, 33, 64, 2, 8), (40, 640, 16, 1, 1), (64 * 17, 8, 128, 1, 2)]


@pytest.mark.parametrize("rows,cols,group,vectors,level", VECTORS)
def test_matvec_small_ring(gpu_small, rows, cols, group, vectors, level):
    g, d = gpu_small, _tile(gpu_small)
    codes, scales, w = _matrix(rows, cols, group, rows)
    qw = g.qweight(codes, scales, rows, group)
    kb, nb = -(-rows // (4 * d)), -(-cols // d)
    x = rand_ct_residues(g, level, 2, vectors * kb, 9)
    ct = g.ct_create(level, 2, vectors * kb, 1)
    g.ct_import(ct, x)
    at = np.unique(np.concatenate([[0, g.N - 1], np.random.default_rng(1).integers(0, g.N, 15)]))
    out = g.matvec_q4(ct, qw, d)
    assert g.ct_meta(out) == (level, 2, vectors * nb, 2)
    operands = [h for k in range(kb * nb) for h in g.encode_q4(qw, d, k, 1, level, diagonal=False)]
    assert np.array_equal(g.ct_export(out)[..., at].astype(object), _operand_sums(g, x, operands, kb, nb, at))


@pytest.mark.parametrize("rows,cols,group,vectors,level", [(768, 384, 128, 1, 1), (1001, 333, 48, 2, 3), (5000, 100, 128, 1, 5), (100, 4500, 64, 1, 0), (512, 130, 32, 5, 12)])
def test_matvec_full_ring(gpu_full, rows, cols, group, vectors, level):
    g, d = gpu_full, 128
    codes, scales, w = _matrix(rows, cols, group, rows)
    qw = g.qweight(codes, scales, rows, group)
    kb, nb = -(-rows // (4 * d)), -(-cols // d)
    x = rand_ct_residues(g, level, 2, vectors * kb, 9)
    ct = g.ct_create(level, 2, vectors * kb, 1)
    g.ct_import(ct, x)
    at = np.unique(np.concatenate([[0, g.N - 1], np.random.default_rng(1).integers(0, g.N, 40)]))
    got = g.ct_export(g.matvec_q4(ct, qw, d))
    operands = g.encode_q4(qw, d, 0, kb * nb, level, diagonal=False)
    assert np.array_equal(got[..., at].astype(object), _operand_sums(g, x, operands, kb, nb, at))


@pytest.mark.parametrize("kb", [8, 9, 127, 129])
def test_matvec_largest_residues(gpu_small, kb):
    """x of all q - 1, on both sides of the counts after which sums are reduced."""
    g = gpu_small
    codes, scales, w = _matrix(4 * kb, 2, 64, kb)
    qw = g.qweight(codes, scales, 4 * kb, 64)
    x = rand_ct_residues(g, 2, 2, kb, 9)
    x[:] = np.array([int(q) - 1 for q in g.primes[:3]], dtype=np.uint64)[None, None, :, None]
    ct = g.ct_create(2, 2, kb, 1)
    g.ct_import(ct, x)
    at = np.array([0, 3, 500, g.N - 1])
    operands = [h for k in range(2 * kb) for h in g.encode_q4(qw, 1, k, 1, 2, diagonal=False)]
    assert np.array_equal(g.ct_export(g.matvec_q4(ct, qw, 1))[..., at].astype(object), _operand_sums(g, x, operands, kb, 2, at))


OTHER_PRIMES = [dict(log_n=10, q_bits=43), dict(log_n=11, q_bits=59), dict(log_n=16, q_bits=44), dict(log_n=16, q0_bits=59), dict(log_n=16, q0_bits=58, q_bits=50, p_bits=58)]


@pytest.mark.parametrize("prm", OTHER_PRIMES)
def test_other_primes(pkg, prm):
    """Primes of other lengths, and 60-bit ones whose transforms take Shoup products; coefficients of the usual size and large ones."""
    g = pkg.open_gpu(pkg.make_params(num_special=3, hamming_weight=32, max_level=3, dnum=3, **prm))
    try:
        d = _tile(g)
        codes, scales, w = _matrix(4 * d + 3, d + 1, 16, 3)
        for factor in (1.0, 2.0**9):
            qw = g.qweight(codes, (scales * np.float32(factor)).astype(np.float32), 4 * d + 3, 16)
            got = g.encode_q4(qw, d, 0, 4, 3)
            for j, b in np.ndindex(2, 2):
                assert np.array_equal(g.pt_export(got[j * 2 + b]), g.pt_export(g.encode(_slots(factor * w, d, b, j, True, g.slots), 3))), (factor, j, b)
        x = rand_ct_residues(g, 3, 2, 6, 9)
        x[:2] = np.array([int(q) - 1 for q in g.primes[:4]], dtype=np.uint64)[None, None, :, None]
        ct = g.ct_create(3, 2, 6, 1)
        g.ct_import(ct, x)
        at = np.unique(np.concatenate([[0, g.N - 1], np.random.default_rng(1).integers(0, g.N, 15)]))
        operands = g.encode_q4(qw, d, 0, 4, 3, diagonal=False)
        assert np.array_equal(g.ct_export(g.matvec_q4(ct, qw, d))[..., at].astype(object), _operand_sums(g, x, operands, 2, 2, at))
    finally:
        g.close()


def test_recorded_encoding_and_matvec(gpu_small):
    """Neither copies from the host, so both can be recorded; the weights are kept as they were."""
    g, d = gpu_small, _tile(gpu_small)
    codes, scales, w = _matrix(100, 33, 16, 4)
    qw = g.qweight(codes, scales, 100, 16)
    x = g.ct_create(2, 2, 2, 1)
    g.ct_import(x, rand_ct_residues(g, 2, 2, 2, 1))
    run = lambda: (g.encode_q4(qw, d, 0, 3, 2), g.matvec_q4(x, qw, d))
    run()
    g.graph_begin()
    pts, out = run()
    graph = g.graph_end()
    res = rand_ct_residues(g, 2, 2, 2, 5)
    g.ct_import(x, res)
    g.graph_launch(graph)
    g.sync()
    now = run()
    assert np.array_equal(g.ct_export(out), g.ct_export(now[1]))
    assert all(np.array_equal(g.pt_export(a), g.pt_export(b)) for a, b in zip(pts, now[0]))


def test_refusals(pkg, gpu_small, gpu_mid):
    g, d = gpu_small, _tile(gpu_small)
    codes, scales, w = _matrix(100, 33, 16, 4)
    for bad in (dict(codes=codes[:-1]), dict(scales=scales[:-1]), dict(rows=98), dict(group=14), dict(rows=0), dict(group=0), dict(codes=codes.astype(np.int8)), dict(scales=scales.astype(np.float64)),
                dict(codes=codes[0])):
        with pytest.raises(ValueError):
            g.qweight(**(dict(codes=codes, scales=scales, rows=100, group=16) | bad))
    for v in (np.nan, np.inf, -np.inf):
        s = scales.copy()
        s[3, 2] = v
        with pytest.raises(pkg.HBError) as e:
            g.qweight(codes, s, 100, 16)
        assert e.value.code == -1
    out = C.c_void_p()
    p, q = codes.ctypes.data_as(C.POINTER(C.c_uint8)), scales.ctypes.data_as(C.POINTER(C.c_float))
    f = g.dll.hb_qweight_create
    assert f(g.ctx, None, q, 100, 33, 16, C.byref(out)) == -1 and f(g.ctx, p, None, 100, 33, 16, C.byref(out)) == -1
    assert f(g.ctx, p, q, 0, 33, 16, C.byref(out)) == -3 and f(g.ctx, p, q, 100, 0, 16, C.byref(out)) == -3 and f(g.ctx, p, q, 100, 33, 0, C.byref(out)) == -3
    qw = g.qweight(codes, scales, 100, 16)
    m = [C.c_int() for _ in range(3)]
    assert g.dll.hb_qweight_meta(qw.ptr, *[C.byref(k) for k in m]) == 0 and [k.value for k in m] == [100, 33, 16]
    for args, code in (((d, 0, 7, 2), -1), ((d, -1, 1, 2), -1), ((d, 0, 0, 2), -1), ((d, 6, 1, 2), -1), ((d, 0, 1, 9), -2), ((d, 0, 1, -1), -2), ((0, 0, 1, 2), -3), ((d + 1, 0, 1, 2), -3), ((1 << 20, 0, 1, 2), -3)):
        with pytest.raises(pkg.HBError) as e:
            g.encode_q4(qw, *args)
        assert e.value.code == code, args
    x = g.ct_create(2, 2, 2, 1)
    for ct, kw, code in ((g.ct_create(2, 2, 3, 1), {}, -3), (g.ct_create(2, 3, 2, 1), {}, -3), (g.ct_create(2, 2, 2, 2), {}, -3), (gpu_mid.ct_create(2, 2, 2, 1), {}, -1), (x, dict(tile=d + 1), -3)):
        with pytest.raises(pkg.HBError) as e:
            g.matvec_q4(ct, qw, **(dict(tile=d) | kw))
        assert e.value.code == code
    with pytest.raises(pkg.HBError):
        gpu_mid.matvec_q4(gpu_mid.ct_create(2, 2, 1, 1), qw, _tile(gpu_mid))
    assert g.dll.hb_matvec_q4(g.ctx, None, qw.ptr, C.c_int(d), C.byref(out)) == -1 and g.dll.hb_matvec_q4(g.ctx, x.ptr, None, C.c_int(d), C.byref(out)) == -1
    g.graph_begin()
    try:
        with pytest.raises(pkg.HBError):
            g.qweight(codes, scales, 100, 16)
    finally:
        g.graph_end()
