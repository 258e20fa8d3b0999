"""BF16 x FP4 products, the sums: partial sums that the CTAs of a cluster exchange, and how closely FP32 sums are held."""
import pytest
import torch

import deepgemm_amd_b200 as dg
from test_bf16_fp4_gpu import check_product, form, make_rows, make_weights, pack_scales  # noqa: F401  (form: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m,n,k", [(128, 1280, 4096), (128, 2560, 4096), (100, 3328, 8192)])
def test_clusters_that_take_several_items(m, n, k):
    """More blocks of D than clusters run at once: every cluster exchanges the partial sums of one block after the other through the same words.
    (All few-row variants cut K into slices for at least one of the sizes, as their cost estimate has it on 148 SMs.)"""
    codes, e, w = make_weights((n, k), 32, 200)
    sf, a = pack_scales(e), make_rows(m, k, 201)
    first = None
    for _ in range(5):
        d = torch.full((m, n), float("nan"), dtype=torch.float, device="cuda")
        dg.bf16_fp4_gemm_nt(a, (codes, sf), d)
        assert first is None or torch.equal(first, d)
        first = d
    check_product(first, a, w)
    assert dg.kernel_status() == 0
