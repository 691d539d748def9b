"""What the Python layer checks of its arguments before it calls the library: with a stand-in for the library."""
from types import SimpleNamespace

import numpy as np
import pytest


def _hemmer(pkg, **lib):
    h = object.__new__(pkg.Hemmer)
    h.lib = SimpleNamespace(slots=512, L=8, **lib)  # tiles of 16: K-groups of 64 rows
    return h


@pytest.mark.parametrize("rows", [64, 1, 0, 129, 1000])
def test_operands_of_a_matrix_of_other_rows(pkg, rows):
    """Blocks are numbered by the matrix's own rows: by others, columns would get the K-groups of their neighbours."""
    calls = []
    h = _hemmer(pkg, qweight_meta=lambda w: (100, 40, 16), encode_q4=lambda *a: calls.append(a) or [None] * a[3])
    with pytest.raises(ValueError):
        h.encode_diagonal_to_row4_q4(None, rows, 40)
    assert not calls


@pytest.mark.parametrize("rows,cols,tiles", [(100, 40, 3), (128, 48, 3), (65, 33, 3), (100, 32, 2)])
def test_operands_of_as_many_blocks(pkg, rows, cols, tiles):
    calls = []
    h = _hemmer(pkg, qweight_meta=lambda w: (100, 40, 16), encode_q4=lambda *a: calls.append(a) or [None] * a[3])
    got = h.encode_diagonal_to_row4_q4(None, rows, cols)
    assert len(got) == tiles and all(len(row) == 2 for row in got) and calls[0][2:4] == (0, 2 * tiles)


def _vectors(pkg, cols):
    """(layer, calls): 100 x 40 matrices, two K-groups of 64 rows and three column tiles"""
    calls = []
    h = _hemmer(pkg, qweight_meta=lambda w: (100, cols, 16), encrypt_many=lambda msgs, level, nonces: len(msgs), ct_meta=lambda ct: (3, 2, ct, 1),
                decrypt_many=lambda members: np.zeros((len(members), 512), dtype=complex))
    h._call = lambda name, x, w: calls.append(name) or 6
    return h, calls


class _Ct(int):
    ptr = None


def test_vectors_of_another_length(pkg):
    """Two vectors of 60 entries are two members, which a matrix of 100 rows would take for one vector of 100; one of 200 are four, two vectors of it."""
    h, calls = _vectors(pkg, 40)
    w = SimpleNamespace(ptr=None)
    for x in (np.ones((2, 60)), np.ones((1, 200)), np.ones((4, 1))):
        ct = h.encrypt_vectors(x, 3, None)
        ct.ct = _Ct(ct.ct)
        with pytest.raises(pkg.HBError):
            h.matvec_q4(ct, w)
    assert not calls
    for x in (np.ones((2, 100)), np.ones((1, 70)), np.ones((3, 128))):
        ct = h.encrypt_vectors(x, 3, None)
        ct.ct = _Ct(ct.ct)
        h.matvec_q4(ct, w)
    h.matvec_q4(pkg.CtxtTensor(_Ct(2), 16, 16, 32), w)  # made another way: the library counts its members
    assert len(calls) == 4


def test_results_of_another_width(pkg):
    """Six members: two vectors of three column tiles, not three of two."""
    h, _ = _vectors(pkg, 40)
    y = h.matvec_q4(pkg.CtxtTensor(_Ct(4), 16, 16, 32), SimpleNamespace(ptr=None))
    for cols in (32, 16, 1, 96):
        with pytest.raises(ValueError):
            h.decrypt_vectors(y, cols)
    assert h.decrypt_vectors(y, 40).shape == (2, 40) and h.decrypt_vectors(pkg.CtxtTensor(6, 16, 16, 32), 32).shape == (3, 32)


def _weights(tiles, groups):
    return [[SimpleNamespace(ct=SimpleNamespace(ptr=SimpleNamespace(value=1)), width=32, shape=(16, 16, 32)) for _ in range(groups)] for _ in range(tiles)]


@pytest.mark.parametrize("sizes,weights", [([0, 0], [None, None]), ([], []), ([1], [_weights(2, 1), _weights(2, 1)]), ([1, 0], [_weights(2, 1)]), ([1], [[]]), ([1], [[[]]])])
def test_experts_without_inputs_or_weights(pkg, sizes, weights):
    """As many lists of weights as sizes, one of them with positions and with weights."""
    calls = []
    h = _hemmer(pkg, matmul_acc_grouped=lambda *a, **k: calls.append(a))
    with pytest.raises(ValueError):
        h.matmul_reuse_experts(None, 2, sizes, weights)
    assert not calls
    h.matmul_reuse_experts(None, 2, [0, 2], [None, _weights(2, 1)])
    assert len(calls) == 1


def test_an_expert_with_an_empty_list(pkg):
    lib = object.__new__(pkg.capi.Lib)
    with pytest.raises(ValueError):
        lib.matmul_acc_grouped(None, 2, [1], [[]], 8)


@pytest.mark.parametrize("far", [2**32, 2**32 + 1, 2**31, -2**31 - 1])
def test_whole_numbers_beyond_32_bits(pkg, far):
    """ctypes drops the bits that do not fit: input 2^32 would be input 0, a group of 2^32 + 1 rows one of a single row, whose scales are not there."""
    calls = []
    lib = object.__new__(pkg.capi.Lib)
    lib._fn = lambda name: lambda *a: calls.append(name) or 0
    lib._op = lambda name, *a: calls.append(name)
    lib.ctx, lib.alive = None, False
    x = SimpleNamespace(ptr=SimpleNamespace(value=None))
    w, codes, scales = [[x]], np.zeros((2, 3), dtype=np.uint8), np.zeros((1, 3), dtype=np.float32)
    for call in (lambda n: lib.matmul_acc_grouped(x, 2, [1], [w], 8, order=[n]), lambda n: lib.matmul_acc_grouped(x, n, [1], [w], 8), lambda n: lib.matmul_acc_grouped(x, 2, [n], [w], 8),
                 lambda n: lib.tensor_acc_cross(x, x, n), lambda n: lib.tensor_acc_cross(x, x, 1, heads=n), lambda n: lib.matvec_q4(x, x, n), lambda n: lib.encode_q4(x, n, 0, 1, 1),
                 lambda n: lib.encode_q4(x, 1, n, 1, 1), lambda n: lib.encode_q4(x, 1, 0, 1, n), lambda n: lib.qweight(codes, scales, 4, abs(n))):
        with pytest.raises(ValueError):
            call(far)
        assert not calls


@pytest.mark.parametrize("far", [2**32 + 1, 2**31])
def test_heads_and_tiles_beyond_32_bits(pkg, far):
    calls = []
    h = _hemmer(pkg)
    h._call = lambda name, *a: calls.append(name)
    t = pkg.CtxtTensor(SimpleNamespace(ptr=None), 16, 16, 32)
    for call in (lambda: h.cross_matmul(t, t, heads=far), lambda: h.cross_matmul(t, t, inner=far), lambda: h.cross_matmul(t, t, target_level=far), lambda: h.cross_scores(t, t, heads=far),
                 lambda: h.cross_scores(t, t, target_level=far)):
        with pytest.raises(ValueError):
            call()
    assert not calls
    h.cross_matmul(t, t), h.cross_scores(t, t)
    assert len(calls) == 2
