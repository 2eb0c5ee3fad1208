"""Sizes that reach every launch shape of ``ravel_matmul`` in every direction, with several chunks of the sum and ragged
last tiles: rows, k and outputs of a Linear, and the shapes (CTAs per product, columns, CTAs that divide k) of y, d x and
d W on a device of 148 SMs."""
from __future__ import annotations

import ctypes

PAIR256, PAIR128, ONE128, ONE64, ONE32, SPLIT2, SPLIT4 = ((2, 256, 1), (2, 128, 1), (1, 128, 1), (1, 64, 1), (1, 32, 1),
                                                          (1, 128, 2), (1, 128, 4))
CASES = [
    ((337, 344, 40), ONE32, ONE64, ONE64),
    ((300, 2056, 2000), ONE64, ONE64, ONE128),
    ((24, 2048, 8192), ONE64, SPLIT4, ONE128),
    ((142, 330, 4976), ONE128, SPLIT4, ONE128),
    ((40, 4864, 5024), SPLIT2, SPLIT2, ONE128),
    ((24, 4509, 5023), SPLIT2, SPLIT2, ONE128),
    ((24, 8192, 512), SPLIT4, ONE64, ONE128),
    ((24, 3888, 41), SPLIT4, ONE64, ONE64),
    ((344, 10064, 41), SPLIT4, ONE128, ONE128),
    ((4608, 4560, 48), ONE32, ONE128, SPLIT2),
    ((4603, 4560, 41), ONE32, ONE128, SPLIT2),
    ((9704, 856, 72), PAIR128, ONE128, SPLIT4),
    ((9703, 853, 70), PAIR128, ONE128, SPLIT4),
    ((856, 5080, 136), SPLIT4, ONE128, PAIR128),
    ((9700, 72, 836), ONE128, PAIR128, SPLIT4),
    ((7112, 336, 4448), PAIR256, PAIR128, PAIR128),
    ((7108, 331, 4443), PAIR256, PAIR128, PAIR128),
    ((136, 9488, 7232), PAIR128, PAIR256, PAIR256),
    ((10431, 6044, 1221), PAIR256, PAIR128, PAIR256),
]
# one row: k, outputs, warps per weight row
ROWS = [(4096, 4096, 1), (4099, 4096, 1), (4096, 2048, 2), (4099, 2047, 2), (4096, 700, 4), (8200, 700, 4), (4096, 72, 8),
        (9000, 41, 8), (64, 700, 1)]


def plan(lib, M, N, K, b_mn):
    """The launch shape of an M x N product over K (``ravel_matmul_plan``)."""
    out = (ctypes.c_int * 3)()
    assert lib.ravel_matmul_plan(M, N, K, b_mn, out) == 0
    return tuple(out)


def plans(lib, M, K, N):
    """Those of y, d x and d W."""
    return plan(lib, M, N, K, 0), plan(lib, M, K, N, 1), plan(lib, N, K, M, 1)
