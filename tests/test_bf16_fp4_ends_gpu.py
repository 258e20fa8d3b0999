"""Ragged BF16 x FP4 products whose ends go back or leave the rows of A: every row belongs to one group or to none."""
import pytest
import torch

import deepgemm_amd_b200 as dg
from test_bf16_fp4_ends_cpu import groups_of
from test_bf16_fp4_gpu import check_product, form, make_rows, make_weights, pack_scales  # noqa: F401  (form: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("rows,ends", [(10, [5, 3, 10]), (400, [200, 17, 399]), (900, [0, 500, 450, 3, 650, -2, 640, 800]), (130, [64, 131, 0, 500]),
                                       (700, [500] + [490 - 12 * i for i in range(40)] + [600]), (300, [20 * (i // 2) if i % 3 else 0 for i in range(70)])])
def test_ends_that_go_back(rows, ends):
    """An end below an earlier one is that one: the group is empty, and the next one begins where the rows given out so far end.  More than 32 groups: also
    across the window of ends that a warp holds."""
    n, k = 264, 512
    codes, e, w = make_weights((len(ends), n, k), 32, 220)
    sf, a = pack_scales(e), make_rows(rows, k, 221)
    d = torch.full((rows, n), -7.0, dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    behind = 0
    for g, (first, count) in enumerate(groups_of(ends, rows)):
        if count:
            check_product(d[first:first + count], a[first:first + count], w[g])
        behind = first + count
    assert (d[behind:] == -7.0).all()
    assert dg.kernel_status() == 0
