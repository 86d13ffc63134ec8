"""How linear_cross_entropy cuts its rows into pieces, at the sizes that it accepts (host arithmetic of the extension)."""
import pytest

from supergrok15_b200 import _build

CAP = 256 << 20


@pytest.mark.parametrize("elem", [2, 4])
@pytest.mark.parametrize("train", [True, False])
def test_pieces_stay_in_bounds(elem, train):
    C = _build.require()
    for V in (1, 2, 8, 9, 64, 127, 129, 1000, 32000, 128000, 1 << 20, (1 << 22) - 1):
        per = 64 if elem == 2 else 4
        ldu = (V + per - 1) // per * per
        for rows in (1, 255, 256, 257, 8188, 65536, 65537, 1 << 23, (1 << 23) + 1, (1 << 30) - 1):
            piece = C.lce_piece_rows(rows, ldu, elem, train)
            assert 1 <= piece <= rows or piece <= (rows + 255) // 256 * 256
            assert piece == rows or piece % 256 == 0
            assert (piece + 127) // 128 <= 65535                           # tile rows are the second dimension of a grid
            bytes_per_row = ldu * elem if train else (V + 127) // 128 * 8  # the exponentials, or a reference and a sum per tile of columns
            assert piece <= 256 or piece * bytes_per_row <= CAP, (V, rows, piece)


def test_ordinary_sizes_are_one_piece():
    C = _build.require()
    assert C.lce_piece_rows(4096, 32000, 2, True) == 4096 and C.lce_piece_rows(65536, 4096, 4, False) == 65536
    assert C.lce_piece_rows(8188, 32000, 2, True) == 4096
