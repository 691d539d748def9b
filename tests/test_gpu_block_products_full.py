"""Products of a transformer block beyond one tile on the ring with 2^16 coefficients, whose tiles have 128 rows and columns: decrypted, against products in 64 bits.

Decrypted values may be off by 2^-14, the bound that every decrypted product of this repository is held to; sums over r tiles by r times that."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -14
D = 128


@pytest.fixture(scope="module")
def ring(pkg):
    """A context of its own: the methods add rotation keys, which tests of missing ones must not find."""
    g = pkg.open_gpu()
    g.keygen()
    yield g
    g.close()


@pytest.fixture(scope="module", params=[0, 1, 2])
def hemmer(request, pkg, ring):
    h = pkg.open_hemmer(ring)
    h.set_schedule(request.param)
    yield h
    h.close()


def _pairs(rng, count):
    return [(rng.uniform(-1, 1, (D, D)), rng.uniform(-1, 1, (D, D))) for _ in range(count)]


def _encrypt(h, pairs, base):
    return h.encrypt2_many(pairs, [base + k for k in range(len(pairs))])


def _halves(h, t):
    z = h.lib.decrypt_many([(t.ct, k) for k in range(h.lib.ct_meta(t.ct)[2])]).real.reshape(-1, D, 2 * D)
    return z[:, :, :D], z[:, :, D:]


@pytest.mark.parametrize("heads,nq,nk", [(2, 1, 3), (1, 3, 2)])
def test_cross_scores(hemmer, heads, nq, nk):
    h, rng = hemmer, np.random.default_rng(nq)
    q, k = _pairs(rng, heads * nq), _pairs(rng, heads * nk)
    got = h.cross_scores(_encrypt(h, q, 100), _encrypt(h, k, 500), heads=heads)
    assert h.lib.ct_meta(got.ct)[:3] == (4, 2, heads * nq * nk)
    for half, z in enumerate(_halves(h, got)):
        for j, hd, i in np.ndindex(nk, heads, nq):
            assert np.abs(z[(j * heads + hd) * nq + i] - q[hd * nq + i][half] @ k[hd * nk + j][half].T).max() < TOL, (half, j, hd, i)


@pytest.mark.parametrize("heads,nq,nk,inner", [(1, 2, 1, 4), (2, 1, 2, 2)])
def test_cross_matmul_sums(hemmer, heads, nq, nk, inner):
    h, rng = hemmer, np.random.default_rng(inner)
    a, b = _pairs(rng, inner * heads * nq), _pairs(rng, inner * heads * nk)
    got = h.cross_matmul(_encrypt(h, a, 100), _encrypt(h, b, 500), heads=heads, inner=inner, target_level=3)
    for half, z in enumerate(_halves(h, got)):
        for j, hd, i in np.ndindex(nk, heads, nq):
            want = sum(a[(r * heads + hd) * nq + i][half] @ b[(r * heads + hd) * nk + j][half] for r in range(inner))
            assert np.abs(z[(j * heads + hd) * nq + i] - want).max() < inner * TOL, (half, j, hd, i)


@pytest.mark.parametrize("rows,cols,group,vectors,level", [(768, 768, 64, 1, 1), (1001, 333, 48, 3, 4)])
def test_vectors_times_4_bit_matrices(hemmer, rows, cols, group, vectors, level):
    h, rng = hemmer, np.random.default_rng(rows)
    code, scales = rng.integers(0, 16, (2 * -(-rows // 2), cols)).astype(np.uint8), rng.uniform(0.002, 0.006, (-(-rows // group), cols)).astype(np.float32)
    w = (code[:rows].astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), group, 0)[:rows]
    x = rng.uniform(-1, 1, (vectors, rows))
    ct = h.encrypt_vectors(x, level, [900 + k for k in range(vectors * -(-rows // (4 * D)))])
    y = h.matvec_q4(ct, h.lib.qweight(code[0::2] | (code[1::2] << 4), scales, rows, group))
    assert h.lib.ct_meta(y.ct)[0] == level - 1
    assert np.abs(h.decrypt_vectors(y, cols) - x @ w).max() < TOL
