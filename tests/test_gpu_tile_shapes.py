"""Products of tiles with tiles of another number, for tiles of every shape: those that are multiplied, against products in 64 bits, and those that are refused.

Decrypted values may be off by 2^-14, the bound that every decrypted product of this repository is held to."""
import ctypes as C
import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -14
SIDES = (8, 16, 32)


@pytest.fixture(scope="module", params=[0, 1, 2])
def hemmer(request, pkg, gpu_mid):
    h = pkg.open_hemmer(gpu_mid)
    h.set_schedule(request.param)
    yield h
    h.close()


def _tensor(pkg, h, tiles, width, nonce):
    """Tiles side by side, at the first and at the middle column of rows of `width` slots."""
    z = np.zeros((h.lib.slots // width, width), dtype=np.complex128)
    for t, at in zip(tiles, (0, width // 2)):
        z[: t.shape[0], at:at + t.shape[1]] = t
    return pkg.CtxtTensor(h.lib.encrypt(h.lib.encode(z.reshape(-1), h.lib.L), nonce), *tiles[0].shape, width)


def _tiles(h, t, rows, cols, count):
    z = h.lib.decrypt(t.ct).real.reshape(-1, t.width)
    return [z[:rows, at:at + cols] for at in (0, t.width // 2)[:count]]


def _products(rows, inner, cols, width, count):
    rng = np.random.default_rng(rows + 100 * inner + 10000 * cols + width)
    a, b = [rng.uniform(-1, 1, (rows, inner)) for _ in range(count)], [rng.uniform(-1, 1, (inner, cols)) for _ in range(count)]
    return a, b, [x @ y for x, y in zip(a, b)]


@pytest.mark.parametrize("inner", SIDES)
def test_sides_up_to_the_inner_one(pkg, hemmer, inner):
    h = hemmer
    for rows, cols in itertools.product([s for s in (1,) + SIDES if s <= inner], repeat=2):
        for width, count in ((inner, 1), (2 * inner, 2)) + (((4 * inner, 2),) if 4 * inner <= 64 else ()):
            a, b, want = _products(rows, inner, cols, width, count)
            got = h.cross_matmul(_tensor(pkg, h, a, width, 1), _tensor(pkg, h, b, width, 2), target_level=2)
            assert got.shape == (rows, cols, width)
            for x, y in zip(_tiles(h, got, rows, cols, count), want):
                assert np.abs(x - y).max() < TOL, (rows, cols, width)


def test_an_inner_side_between_powers_of_two(pkg, hemmer):
    """20 columns against 20 rows in tiles of 32, zeros behind them."""
    h = hemmer
    a, b, want = _products(32, 20, 16, 32, 1)
    got = h.cross_matmul(_tensor(pkg, h, a, 32, 1), _tensor(pkg, h, b, 32, 2), target_level=2)
    assert np.abs(_tiles(h, got, 32, 16, 1)[0] - want[0]).max() < TOL


@pytest.mark.parametrize("rows,inner,cols,width", [(16, 8, 8, 16), (8, 8, 16, 16), (32, 16, 16, 32), (32, 16, 32, 64), (16, 16, 32, 64), (20, 32, 32, 32), (32, 32, 20, 32), (32, 32, 32, 40),
                                                   (32, 32, 32, 16), (64, 64, 64, 64), (20, 20, 20, 40)])
def test_sides_that_no_sum_over_the_inner_one_reaches(pkg, hemmer, rows, inner, cols, width):
    h = hemmer
    a, b = h.lib.ct_create(8, 2, 1, 1), h.lib.ct_create(8, 2, 1, 1)
    with pytest.raises(pkg.HBError) as e:
        h.cross_matmul(pkg.CtxtTensor(a, rows, inner, width), pkg.CtxtTensor(b, inner, cols, width), target_level=2)
    assert e.value.code == -1


@pytest.mark.parametrize("shape", [(0, 8, 8), (8, 0, 8), (8, 8, 0), (-8, 8, 8), (8, 8, -8)])
def test_empty_tiles(pkg, hemmer, shape):
    h = hemmer
    a = h.lib.ct_create(8, 2, 1, 1)
    with pytest.raises(pkg.HBError) as e:
        h.cross_matmul(pkg.CtxtTensor(a, *shape), pkg.CtxtTensor(a, shape[1], shape[0], shape[2]), target_level=2)
    assert e.value.code == -1


@pytest.mark.parametrize("shape", [(16, 32, 32), (4, 8, 8), (1, 16, 16)])
def test_scores_of_a_key_tile_alone_with_fewer_rows(pkg, hemmer, shape):
    h = hemmer
    with pytest.raises(pkg.HBError) as e:
        h.cross_scores(pkg.CtxtTensor(h.lib.ct_create(8, 2, 1, 1), *shape), pkg.CtxtTensor(h.lib.ct_create(8, 2, 1, 1), *shape), target_level=2)
    assert e.value.code == -1


@pytest.mark.parametrize("rows,keys", [(32, 16), (16, 32), (8, 16), (32, 8), (16, 16), (1, 32)])
def test_scores_of_tiles_with_other_numbers_of_rows(pkg, hemmer, rows, keys):
    h, rng = hemmer, np.random.default_rng(rows + keys)
    q, k = [rng.uniform(-1, 1, (rows, 32)) for _ in range(2)], [rng.uniform(-1, 1, (keys, 32)) for _ in range(2)]
    got = h.cross_scores(_tensor(pkg, h, q, 64, 1), _tensor(pkg, h, k, 64, 2), target_level=2)
    assert got.shape == (rows, keys, 64)
    for x, a, b in zip(_tiles(h, got, rows, keys, 2), q, k):
        assert np.abs(x - a @ b.T).max() < TOL


def test_rows_behind_a_shorter_key_tile_are_not_keys(pkg, hemmer):
    """The shape says how many rows are keys, whatever the slots behind them hold."""
    h, rng = hemmer, np.random.default_rng(1)
    q, k = [rng.uniform(-1, 1, (32, 32)) for _ in range(2)], [rng.uniform(-1, 1, (32, 32)) for _ in range(2)]
    whole = _tensor(pkg, h, k, 64, 2)
    got = h.cross_scores(_tensor(pkg, h, q, 64, 1), pkg.CtxtTensor(whole.ct, 16, 32, 64), target_level=2)
    for x, a, b in zip(_tiles(h, got, 32, 32, 2), q, k):
        assert np.abs(x[:, :16] - a @ b[:16].T).max() < TOL


def test_scores_through_the_entry_with_one_shape(pkg, hemmer):
    h, rng = hemmer, np.random.default_rng(2)
    q, k = (_tensor(pkg, h, [rng.uniform(-1, 1, (16, 32)) for _ in range(2)], 64, n) for n in (1, 2))
    one = h._call("cross_scores", q.ct.ptr, k.ct.ptr, *h._shp(q), C.c_int(1), C.c_int(2))
    assert np.array_equal(h.lib.ct_export(one), h.lib.ct_export(h.cross_scores(q, k, target_level=2).ct))


@pytest.mark.parametrize("query,key", [((32, 32, 64), (32, 16, 64)), ((32, 32, 64), (32, 32, 32)), ((16, 16, 32), (32, 16, 32)), ((32, 32, 64), (20, 32, 64))])
def test_scores_of_tiles_that_do_not_meet(pkg, hemmer, query, key):
    h = hemmer
    with pytest.raises(pkg.HBError) as e:
        h.cross_scores(pkg.CtxtTensor(h.lib.ct_create(8, 2, 1, 1), *query), pkg.CtxtTensor(h.lib.ct_create(8, 2, 1, 1), *key), target_level=2)
    assert e.value.code == -1
