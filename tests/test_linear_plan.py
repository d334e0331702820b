"""Sizes that reach every form of the dense product's tile kernel.

(tile, K split): [plain, swiglu], each (columns in fours on aligned rows, any
columns on rows that are copied first) as (M, N, K).  Rows past the last whole
tile, columns past the last whole block and a partial K step in each.  The rule
that chooses is the library's, asked here on the CPU."""
import os

import pytest

from xtu_moe_amd import _lib
from xtu_moe_amd.linear import ACTIVATIONS

FORMS = {
    (0, False): [((68, 44, 136), (69, 42, 133)),
                 ((75, 44, 136), (68, 42, 135))],
    (0, True): [((72, 44, 1416), (70, 41, 1417)),
                ((67, 44, 1424), (65, 41, 1465))],
    (1, False): [((641, 744, 136), (455, 1041, 133)),
                 ((541, 452, 136), (647, 369, 131))],
    (1, True): [((66, 676, 2648), (66, 685, 2575)),
                ((80, 344, 3384), (68, 346, 3307))],
    (2, False): [((2737, 716, 136), (3594, 519, 135)),
                 ((1391, 740, 136), (1711, 578, 135))],
    (2, True): [((641, 456, 4272), (200, 679, 6447)),
                ((403, 196, 6992), (193, 343, 6443))],
    (3, False): [((3863, 1044, 328), (2321, 1733, 321)),
                 ((647, 4216, 200), (2722, 1101, 193))],
    (3, True): [((710, 2780, 4192), (1474, 1353, 4179)),
                ((3024, 324, 4136), (1730, 578, 4195))],
    (4, False): [((1726, 1172, 736), (1234, 1615, 713)),
                 ((1155, 872, 712), (772, 1258, 713))],
    (4, True): [((836, 1164, 4144), (1602, 582, 4045)),
                ((810, 620, 4104), (1243, 385, 4121))],
    (5, False): [((2482, 4916, 136), (3599, 3333, 139)),
                 ((3634, 1668, 136), (2083, 2898, 133))],
    (5, True): [((1157, 3416, 3688), (2398, 1675, 3623)),
                ((2435, 856, 3640), (1292, 1541, 3591))],
}


def plan(M, N, K, act):
    """(tile, splits) that the library takes, or None for the stream of few rows."""
    r = _lib.load().xtu_linear_plan(M, N, K, ACTIVATIONS[act])
    assert r >= 0
    return None if r == 0 else (r % 256 - 1, r // 256)


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_every_form_is_reached():
    for (tile, split), sides in FORMS.items():
        for gated, sizes in enumerate(sides):
            for vec, (M, N, K) in zip((True, False), sizes):
                assert (N % 4 == 0) == vec and (K % 8 == 0) == vec
                assert M % 64 and N % 16 and K % 64
                for act in ("swiglu",) if gated else ("none", "gelu"):
                    got = plan(M, N, K, act)
                    assert got[0] == tile and (got[1] > 1) == split, (tile, split, M, N, K)


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_plan_of_other_sizes():
    assert plan(1, 512, 2048, "swiglu") is None and plan(16, 256, 3000, "none") is None
    call = _lib.load().xtu_linear_plan
    assert call(0, 1, 1, 0) == call(1, 0, 1, 0) == call(1, 1, 0, 0) == -1
    assert call(-1, 1, 1, 0) == call(1, 1 << 29, 1, 0) == call((1 << 31) - 1, 1, 1, 0) == -1
