"""The ragged layout's ends on the host: what the tile scheduler of the many-row form makes of ends that go back or leave the rows of A."""
import ctypes as C

import pytest

from deepgemm_amd_b200 import _lib


def groups_of(ends, m):
    """(first row, rows) per group: a group begins where the one before it ends; an end counts as the largest up to it, inside [0, m]."""
    at, out = 0, []
    for e in ends:
        end = max(at, min(max(e, 0), m))
        out.append((at, end - at))
        at = end
    return out


@pytest.mark.parametrize("m,ends", [(10, [5, 3, 10]), (700, [300, 20, 0, 300, 129, 640]), (300, [300, 0, 300]), (260, [-4, 130, -1, 131, 90, 9999, 7]), (50, [0, 0, 0]),
                                    (1000, [1000] * 40), (600, [600 - 7 * i for i in range(50)])])
@pytest.mark.parametrize("ctas", [1, 5])
def test_rows_belong_to_one_group(m, ends, ctas):
    n, block_n, seen = 300, 96, []
    for cta in range(ctas):
        out = (C.c_uint32 * 4096)()
        got = _lib.lib.dg_enumerate_tiles(_lib.DG_GEMM_M_GROUPED_RAGGED, block_n, 4, m, n, len(ends), (C.c_int32 * len(ends))(*ends), cta, ctas, out, 1024)
        seen += [tuple(out[4 * i:4 * i + 4]) for i in range(got)]
    want = [(first + 128 * b, j, g, min(128, rows - 128 * b)) for g, (first, rows) in enumerate(groups_of(ends, m)) for b in range(-(-rows // 128)) for j in range(-(-n // block_n))]
    assert sorted(seen) == sorted(want)
