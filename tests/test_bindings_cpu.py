"""What the Python layer checks of its arguments before it calls the library: with a stand-in for the library."""
from types import SimpleNamespace

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
