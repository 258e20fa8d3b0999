"""Calls of the BF16 x FP4 products that the documentation allows, beside the plain ones."""
import pytest
import torch

import deepgemm_amd_b200 as dg
from test_bf16_fp4_gpu import check_product, check_ragged, form, make_rows, make_weights, pack_scales, ragged_case  # noqa: F401  (form: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("n", [1, 3, 9, 129])
@pytest.mark.parametrize("m", [1, 17, 200])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float])
def test_very_few_columns(m, n, out):
    k = 256
    codes, e, w = make_weights((n, k), 32, 260)
    a, wide = make_rows(m, k, 261), torch.full((m, 144), -7.0, dtype=out, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), wide[:, :n])
    check_product(wide[:, :n], a, w)
    assert (wide[:, n:] == -7.0).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("counts", [[2, 0, 1], [40, 1, 0, 150]])
def test_ragged_with_very_few_columns(counts):
    n, k = 3, 256
    codes, e, w, a, ends = ragged_case(counts, 2, n, k, 32, 262)
    wide = torch.full((a.size(0), 8), -7.0, dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), wide[:, :n], ends)
    check_ragged(wide[:, :n], a, w, counts, -7.0)
    assert (wide[:, n:] == -7.0).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("counts", [[3, 0, 5, 1], [70, 9, 0, 130]])
def test_rows_behind_the_groups_and_in_other_groups_do_not_reach_a_group(counts):
    """A group full of infinities and NaN, and such rows behind the last one: they share tiles and slots with their neighbours, and no results."""
    n, k, bad = 264, 512, 1 if counts[1] else 2
    codes, e, w, a, ends = ragged_case(counts, 5, n, k, 32, 263)
    first = sum(counts[:bad])
    a[first:first + counts[bad]] = float("inf")
    a[sum(counts):] = float("nan")
    d = torch.full((a.size(0), n), -7.0, dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends)
    start = 0
    for g, c in enumerate(counts):
        if g == bad:
            assert not torch.isfinite(d[start:start + c].float()).any()
        elif c:
            check_product(d[start:start + c], a[start:start + c], w[g])
        start += c
    assert (d[start:] == -7.0).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("rows", [12, 300])
def test_fp32_scales_by_group_and_in_a_graph(rows):
    """FP32 scales are packed on the fly into a tensor of the call's own; the recipe may be a list, the ends a slice of a longer tensor."""
    n, k, gran, groups = 264, 640, 128, 3
    codes, e, w = make_weights((groups, n, k), gran, 264)
    a, scales = make_rows(rows, k, 265), torch.exp2(e.float() - 127)
    ends = torch.tensor([0, 0, rows // 3, rows // 3, rows], dtype=torch.int32, device="cuda")[2:]
    d, d2 = (torch.full((rows, n), -7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends, recipe_b=(1, gran))
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, scales), d2, ends, recipe_b=[1, gran])
    assert torch.equal(d, d2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, scales), d2, ends, recipe_b=(1, gran))
        dg.bf16_fp4_gemm_nt(a, (codes[1], scales[1]), d, recipe_b=(1, gran))
    for seed in (266, 267):
        a.copy_(make_rows(rows, k, seed))
        d.fill_(float("nan"))
        d2.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check_product(d, a, w[1])
        check_product(d2[:rows // 3], a[:rows // 3], w[0])
        check_product(d2[rows // 3:], a[rows // 3:], w[2])


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", [3, 30, 90, 400])
def test_c_as_another_view_of_d(m):
    n, k = 136, 384
    codes, e, w = make_weights((n, k), 32, 268)
    a, wide = make_rows(m, k, 269), torch.randn((m, 160), device="cuda")
    before = wide.clone()
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), wide[:, :n], c=wide[:, :n])
    check_product(wide[:, :n], a, w, added=before[:, :n])
    assert torch.equal(wide[:, n:], before[:, n:])


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("sms", [2, 20, 90])
def test_fewer_sms(sms):
    before = dg.get_num_sms()
    try:
        dg.set_num_sms(sms)
        for m, n, k in ((4, 520, 4096), (30, 1032, 1024), (150, 520, 640), (600, 264, 2304)):
            codes, e, w = make_weights((n, k), 32, 270)
            a, d = make_rows(m, k, 271), torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
            dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
            check_product(d, a, w)
        counts = [3, 0, 70, 131]
        codes, e, w, a, ends = ragged_case(counts, 1, 264, 640, 32, 272)
        d = torch.full((a.size(0), 264), -7.0, dtype=torch.bfloat16, device="cuda")
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends)
        check_ragged(d, a, w, counts, -7.0)
    finally:
        dg.set_num_sms(before)
    assert dg.kernel_status() == 0
