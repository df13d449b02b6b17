"""The grouped products' choice of tiles (ml_grouped_matmul_plan, host arithmetic): the products listed in
grouped_plans.py, which the GPU tests run, reach every tile of the ring kernel, in each storage order, with whole
tiles and with tiles in parts, so a change of the choice cannot leave a form untested."""
import ctypes
import os

import pytest

pytest.importorskip("torch")

import grouped_plans as gp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mask_loss_amd", "libmask_loss_hip.so")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    return gp.declare(ctypes.CDLL(LIB))


@pytest.mark.parametrize("case", range(len(gp.CASES)))
def test_listed_products_take_their_tile(lib, case):
    dtype, tile, way, merged, *call = gp.CASES[case]
    p = gp.plan_of(lib, dtype, *call)
    assert p.ring and (p.tile_rows, p.tile_columns) == tile and bool(p.merged) == merged
    ways = gp.how(p, *call)
    assert way in ways if way != "whole" else ways == {"whole"}
    rows, K, N, _, matrices, product, _ = call
    reduced = {gp.FORWARD: K, gp.INPUT: N, gp.WEIGHT: rows // matrices}[product]
    stage = p.stage_bytes // (4 if dtype == gp.F32 else 2)
    assert reduced >= 4 * stage and (product == gp.WEIGHT or reduced % stage)


def test_every_form_is_listed():
    """Tiles x (reduced index contiguous in the matrix or by rows, weight gradient) x whole and in parts."""
    forms = set()
    for dtype, tile, way, merged, *_, product, transposed in gp.CASES:
        kind = "weight" if product == gp.WEIGHT else "contiguous" if (product == gp.FORWARD) == transposed else "rows"
        forms.add((dtype, tile, kind, "whole" if way == "whole" else "parts", merged))
    want = {(dtype, tile, kind, way, merged)
            for dtype, tiles in ((gp.BF16, ((128, 128), (128, 256), (256, 256))), (gp.F32, ((128, 128),)))
            for tile in tiles for kind in ("weight", "contiguous", "rows") for way in ("whole", "parts")
            for merged in ((False,) if kind == "weight" else (False, True))}
    assert want == forms


def test_other_plans(lib):
    """Few rows per group and rows off 16-byte boundaries: one workgroup per tile."""
    p = gp.plan_of(lib, gp.BF16, 64, 1024, 2048, 8, 8, gp.FORWARD, True)
    assert (p.ring, p.tile_rows, p.tile_columns) == (0, 32, 128)
    p = gp.plan_of(lib, gp.BF16, 4096, 1023, 2048, 8, 8, gp.FORWARD, True, aligned=False)
    assert (p.ring, p.tile_rows, p.tile_columns) == (0, 128, 128)


def test_plan_refusals(lib):
    p, s = gp.Plan(), gp.Shape(64, 128, 256, 4, 2)
    ref = ctypes.byref
    for args, words in (((ref(s), gp.BF16, 3, 0, 1, 0, ref(p)), "unknown product"),
                        ((ref(s), gp.BF16, 0, 0, 1, 0, None), "no plan"),
                        ((ref(gp.Shape(64, 127, 256, 4, 2)), gp.BF16, 0, 0, 1, 0, ref(p)), "16-byte"),
                        ((ref(gp.Shape(64, 128, 256, 5, 2)), gp.BF16, 0, 0, 1, 0, ref(p)), "invalid shape"),
                        ((None, gp.BF16, 0, 0, 0, 0, ref(p)), "invalid shape"),
                        ((None, gp.BF16, 0, 0, 1, 0, ref(p)), "16-byte")):
        assert lib.ml_grouped_matmul_plan(*args) == 1
        assert words in lib.ml_last_error().decode()
