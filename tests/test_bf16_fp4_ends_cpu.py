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


ENDS = [[0, 0, 5], [1, 2, 3, 4, 5, 6, 7, 8], [130, 130, 131, 194, 451], [64, 129, 257, 386, 386], [0, 0, 0], [1000], [5, 3, 10], [700, 20, 701], [63, 64, 65, 66, 130, 4000]]


@pytest.mark.parametrize("ends", ENDS + [[3 * (i + 1) for i in range(70)]], ids=str)
@pytest.mark.parametrize("block_m", [64, 128])
@pytest.mark.parametrize("ctas", [1, 6])
def test_tiles_and_slots(ends, block_m, ctas, monkeypatch):
    """Both tile heights: every row of D once, its row of the split A in the slots of its group.  Groups' slots do not meet, begin on multiples of four (where a
    copy of their scale words may) and end inside the workspace: two planes of slots with a scale per 32 elements."""
    n, block_n, k, m = 300, 96, 4096, max(1, min(max(ends), 1200))
    tiles = []
    for cta in range(ctas):
        out = (C.c_uint32 * (5 * 1024))()
        got = _lib.lib.dg_enumerate_ragged_tiles(block_m, block_n, 4, m, n, len(ends), (C.c_int32 * len(ends))(*ends), cta, ctas, out, 1024)
        assert got <= 1024
        tiles += [tuple(out[5 * i:5 * i + 5]) for i in range(got)]
    monkeypatch.setenv("DG_FORCE_BF16_FP4_FORM", "5")          # the form that splits A ahead of the product, whatever the sizes would choose
    args = _lib.GemmArgs()
    args.m, args.n, args.k, args.num_groups, args.d_dtype = m, 4096, k, len(ends), _lib.DG_BF16
    slots = _lib.lib.dg_bf16_fp4_workspace_bytes(C.byref(args), 1) // (2 * (k + k // 32))
    want, taken = [], set()
    for g, (first, rows) in enumerate(groups_of(ends, m)):
        slot = -(-first // 4) * 4 + 4 * g
        mine = set(range(slot, slot + rows))
        assert not taken & mine and slot + rows <= slots
        taken |= mine
        want += [(first + block_m * b, j, g, min(block_m, rows - block_m * b), slot + block_m * b) for b in range(-(-rows // block_m)) for j in range(-(-n // block_n))]
    assert sorted(tiles) == sorted(want) and all(t[4] % 4 == 0 for t in tiles)


@pytest.mark.parametrize("kw", [dict(block_m=32), dict(block_n=0), dict(cta=3), dict(cta=-1), dict(ends=None)], ids=str)
def test_the_walk_refuses(kw):
    a = dict(block_m=64, block_n=96, m=10, ends=(C.c_int32 * 1)(10), cta=0, ctas=3)
    a.update(kw)
    assert _lib.lib.dg_enumerate_ragged_tiles(a["block_m"], a["block_n"], 4, a["m"], 300, 1, a["ends"], a["cta"], a["ctas"], None, 0) < 0
