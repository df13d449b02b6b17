"""Products that take each tile of the grouped products' ring kernel, and what ml_grouped_matmul_plan says of
them: shared by the CPU test of the choice and the GPU test of the results."""
import ctypes

import numpy as np

F32, BF16 = 0, 1
FORWARD, INPUT, WEIGHT = 0, 1, 2

# dtype (float16 is planned as bfloat16), tile, how ("whole": no tile in parts; "parts": parts of the only
# round; "rest": of the last one behind whole rounds; on one XCD at least), merged, rows, K, N, groups,
# matrices, product, transposed.  The reduced length of a forward or d input is four stages or more and not
# a whole number of them; the groups' borders cut a weight gradient's.
CASES = [
    (BF16, (128, 128), "whole", False, 228, 64, 264, 1, 1, 1, False),
    (BF16, (128, 128), "parts", False, 212, 72, 472, 4, 1, 1, False),
    (BF16, (128, 128), "rest", False, 370, 1632, 8256, 8, 8, 0, True),
    (BF16, (128, 128), "whole", True, 200, 280, 64, 20, 2, 0, True),
    (BF16, (128, 128), "parts", True, 203, 72, 488, 20, 2, 1, False),
    (BF16, (128, 128), "rest", True, 373, 1720, 6504, 40, 10, 0, True),
    (BF16, (128, 128), "whole", False, 228, 64, 264, 1, 1, 1, True),
    (BF16, (128, 128), "parts", False, 212, 72, 472, 4, 1, 1, True),
    (BF16, (128, 128), "rest", False, 253, 2160, 16496, 1, 1, 0, False),
    (BF16, (128, 128), "whole", True, 200, 280, 64, 20, 2, 0, False),
    (BF16, (128, 128), "parts", True, 203, 72, 488, 20, 2, 1, True),
    (BF16, (128, 128), "rest", True, 13469, 1480, 528, 6, 3, 0, False),
    (BF16, (128, 128), "whole", False, 396, 64, 64, 1, 1, 2, False),
    (BF16, (128, 128), "parts", False, 457, 64, 64, 1, 1, 2, False),
    (BF16, (128, 128), "rest", False, 14731, 152, 3416, 100, 10, 2, False),
    (BF16, (128, 256), "whole", False, 389, 136, 7560, 8, 8, 0, True),
    (BF16, (128, 256), "parts", False, 1261, 2696, 5672, 6, 6, 1, False),
    (BF16, (128, 256), "whole", True, 592, 152, 5008, 24, 12, 0, True),
    (BF16, (128, 256), "parts", True, 850, 3368, 5720, 24, 6, 1, False),
    (BF16, (128, 256), "whole", False, 396, 184, 4880, 11, 11, 0, False),
    (BF16, (128, 256), "parts", False, 227, 200, 8744, 7, 7, 1, True),
    (BF16, (128, 256), "rest", False, 2723, 1264, 5456, 5, 5, 0, False),
    (BF16, (128, 256), "whole", True, 439, 168, 4872, 24, 12, 0, False),
    (BF16, (128, 256), "parts", True, 325, 256, 5288, 40, 10, 1, True),
    (BF16, (128, 256), "rest", True, 1014, 1032, 12528, 100, 10, 0, False),
    (BF16, (128, 256), "whole", False, 224, 144, 17360, 1, 1, 2, False),
    (BF16, (128, 256), "parts", False, 13548, 952, 64, 1, 1, 2, True),
    (BF16, (128, 256), "rest", False, 990, 272, 46040, 4, 1, 2, False),
    (BF16, (256, 256), "whole", False, 257, 528, 4408, 7, 7, 0, True),
    (BF16, (256, 256), "parts", False, 16390, 3800, 144, 4, 4, 0, True),
    (BF16, (256, 256), "rest", False, 12877, 1328, 1208, 5, 5, 0, True),
    (BF16, (256, 256), "whole", True, 311, 3392, 520, 18, 9, 1, False),
    (BF16, (256, 256), "parts", True, 16049, 136, 3816, 32, 8, 1, False),
    (BF16, (256, 256), "rest", True, 8003, 2048, 1176, 6, 3, 1, False),
    (BF16, (256, 256), "whole", False, 257, 528, 4408, 7, 7, 0, False),
    (BF16, (256, 256), "parts", False, 512, 240, 21008, 1, 1, 1, True),
    (BF16, (256, 256), "rest", False, 16238, 920, 736, 4, 4, 1, True),
    (BF16, (256, 256), "whole", True, 311, 3392, 520, 18, 9, 1, True),
    (BF16, (256, 256), "parts", True, 16787, 3064, 144, 10, 5, 0, False),
    (BF16, (256, 256), "rest", True, 3117, 808, 5096, 8, 2, 0, False),
    (BF16, (256, 256), "whole", False, 209, 136, 36856, 1, 1, 2, False),
    (BF16, (256, 256), "parts", False, 2111, 160, 16640, 2, 1, 2, False),
    (BF16, (256, 256), "rest", False, 1494, 136, 33648, 2, 2, 2, False),
    (F32, (128, 128), "whole", False, 201, 136, 64, 4, 1, 0, True),
    (F32, (128, 128), "parts", False, 205, 72, 232, 1, 1, 1, False),
    (F32, (128, 128), "rest", False, 376, 368, 6384, 10, 10, 0, True),
    (F32, (128, 128), "whole", True, 221, 136, 64, 20, 2, 0, True),
    (F32, (128, 128), "parts", True, 230, 64, 232, 4, 2, 1, False),
    (F32, (128, 128), "rest", True, 353, 376, 6976, 100, 10, 0, True),
    (F32, (128, 128), "whole", False, 201, 136, 64, 4, 1, 0, False),
    (F32, (128, 128), "parts", False, 205, 72, 232, 1, 1, 1, True),
    (F32, (128, 128), "rest", False, 376, 368, 6384, 10, 10, 0, False),
    (F32, (128, 128), "whole", True, 221, 136, 64, 20, 2, 0, False),
    (F32, (128, 128), "parts", True, 230, 64, 232, 4, 2, 1, True),
    (F32, (128, 128), "rest", True, 353, 376, 6976, 100, 10, 0, False),
    (F32, (128, 128), "whole", False, 224, 64, 64, 8, 2, 2, False),
    (F32, (128, 128), "parts", False, 262, 64, 64, 2, 1, 2, False),
    (F32, (128, 128), "rest", False, 4646, 136, 2728, 48, 12, 2, False),
]


class Shape(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int64) for k in ["rows", "K", "N", "groups", "matrices"]]


class Plan(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int32) for k in ["tile_rows", "tile_columns", "ring", "stage_bytes", "workgroups", "parts",
                                              "fewest_parts", "merged"]]


def declare(lib):
    lib.ml_grouped_matmul_plan.argtypes = [ctypes.POINTER(Shape)] + [ctypes.c_int] * 5 + [ctypes.POINTER(Plan)]
    lib.ml_last_error.restype = ctypes.c_char_p
    return lib


def plan_of(lib, dtype, rows, K, N, groups, matrices, product, transposed, aligned=True, equal=False):
    p = Plan()
    rc = lib.ml_grouped_matmul_plan(ctypes.byref(Shape(rows, K, N, groups, matrices)), dtype, product, transposed,
                                    aligned, equal, ctypes.byref(p))
    assert rc == 0, lib.ml_last_error()
    return p


def counts_of(rows, groups):
    """Rows of the groups, of a case that leaves one row before the first and two behind the last."""
    return np.random.default_rng(rows + groups).multinomial(rows - 3, np.ones(groups) / groups)


def how(p, rows, K, N, groups, matrices, product, transposed):
    """Ways in which the XCDs' last tiles are made, from the rule that the kernels apply to the counts: each XCD
    takes a run of consecutive tiles, and those that do not fill a round of its workgroups are split where
    there are `fewest_parts` workgroups or more to a tile."""
    if product == WEIGHT:
        m, n = (N, K) if transposed else (K, N)
        tiles = matrices * -(-m // p.tile_rows)
    else:
        n = N if product == FORWARD else K
        counts = counts_of(rows, groups)
        if matrices == 1:
            counts = counts.sum(keepdims=True)
        elif p.merged:
            counts = counts.reshape(-1, matrices).sum(0)
        tiles = sum(-(-int(c) // p.tile_rows) for c in (*counts, 1, 2))
    tiles *= -(-n // p.tile_columns)
    each, turns, ways = -(-tiles // 8), p.workgroups // 8, set()
    for xcd in range(8):
        mine = max(0, min(each, tiles - xcd * each))
        rest = mine % turns
        parts = min(p.parts if mine < turns else min(p.parts, 8), turns // rest) if rest else 1
        split = parts >= (2 if mine < turns else p.fewest_parts)
        ways.add("whole" if not split else "parts" if mine < turns else "rest")
    return ways
