"""The tile that each size takes, without a device: the cases that the GPU tests run by tile (tests/tile_cases.py) take the one that
they are there for, and they take every one that there is."""
import pytest

from test_abi import header_enum, lib  # noqa: F401  (fixture)
from tile_cases import CASES, RAGGED, RAGGED_DW, RAGGED_T, W4, W4_T, rows_of

SMALL, DEEP = (64, 128, 2), (64, 128, 4)
TILES = {W4: {SMALL, (64, 256, 2), (128, 128, 2), (128, 256, 2)}, W4_T: {SMALL, (128, 128, 2), (256, 256, 2), (256, 128, 2)},
         RAGGED: {SMALL, DEEP, (128, 128, 2), (128, 128, 4), (256, 256, 2)}, RAGGED_T: {SMALL, DEEP, (128, 128, 2), (128, 128, 4), (256, 256, 2)},
         RAGGED_DW: {(128, 128, 2), (128, 128, 4), (256, 256, 2)}}


def plan(lib, product, rows, k, n, E):   # noqa: F811
    p = lib.qmm_tile_plan(product, rows, k, n, E)
    return (p >> 16 & 0xFFFF, p & 0xFFFF, p >> 32 & 0xFF, p >> 40) if p > 0 else p


@pytest.mark.parametrize("product,counts,first,tail,n,k,tile", CASES)
def test_cases_take_their_tile(lib, product, counts, first, tail, n, k, tile):   # noqa: F811
    assert plan(lib, product, rows_of(counts, first, tail), k, n, len(counts)) == tile


def test_cases_take_every_tile():
    """Every tile with a whole sum, sums in 2, 4, 8 and 16 parts in each kind of product, and by more experts than one."""
    for product, tiles in TILES.items():
        mine = [c for c in CASES if c[0] == product]
        assert {c[6][:3] for c in mine if c[6][3] == 1} == tiles
        assert {c[6][3] for c in mine} == {1, 2, 4, 8, 16}
        assert any(len(c[1]) > 1 and c[6][3] > 1 for c in mine)


def test_products_and_sizes(lib):   # noqa: F811
    assert header_enum("qmm_product") == {"QMM_PRODUCT_W4": W4, "QMM_PRODUCT_W4_T": W4_T, "QMM_PRODUCT_RAGGED": RAGGED,
                                          "QMM_PRODUCT_RAGGED_T": RAGGED_T, "QMM_PRODUCT_RAGGED_DW": RAGGED_DW}
    assert plan(lib, RAGGED, 4, 64, 64, 2) == 0 and plan(lib, RAGGED, 0, 64, 64, 2) == 0 and plan(lib, W4_T, 0, 64, 64, 1) == 0
    for product in range(5):
        for rows, k, n, E in ((-1, 64, 64, 1), (80, 60, 64, 1), (80, 64, 0, 1), (80, 64, 64, 0), (80, 64, 64, 1025), ((1 << 24) + 1, 64, 64, 1)):
            assert plan(lib, product, rows, k, n, E) == -1
    assert plan(lib, 5, 80, 64, 64, 1) == -1 and plan(lib, -1, 80, 64, 64, 1) == -1
    # parts have their workspace
    for product, counts, first, tail, n, k, tile in CASES:
        rows, E = rows_of(counts, first, tail), len(counts)
        need = {W4: lambda: lib.qmm_w4_mm_workspace_size(rows, k, n, E, 1), W4_T: lambda: lib.qmm_w4_mm_t_workspace_size(rows, k, n, E),
                RAGGED: lambda: lib.qmm_ragged_mm_workspace_size(rows, k, n, E), RAGGED_T: lambda: lib.qmm_ragged_mm_t_workspace_size(rows, k, n, E),
                RAGGED_DW: lambda: lib.qmm_ragged_mm_dw_workspace_size(rows, k, n, E)}[product]()
        outputs = {W4: rows * n, W4_T: rows * k, RAGGED: rows * n, RAGGED_T: rows * k, RAGGED_DW: E * n * k}[product]
        assert need == (4 * outputs * tile[3] if tile[3] > 1 else 0)
