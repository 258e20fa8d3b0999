"""BF16 x FP4 products under the documented tuning settings: the same bits."""
import pytest
import torch

import deepgemm_amd_b200 as dg
from test_bf16_fp4_gpu import check_product, check_ragged, make_rows, make_weights, pack_scales, ragged_case

pytestmark = pytest.mark.gpu

SETTINGS = [{"PRODUCER_WHOLE_WARP": "0"}, {"MMA_WHOLE_WARP": "0"}, {"PRODUCER_WHOLE_WARP": "0", "MMA_WHOLE_WARP": "0"}, {"L2_HINT": "1"}, {"L2_HINT": "2"},
            {"EPILOGUE_BACKOFF_NS": "100"}, {"FORCE_STORE_BUFFERS": "2"}, {"PROFILE": "1"}]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}={v}" for k, v in s.items()))
def test_the_gemm_form_gives_the_same_bits(settings, monkeypatch):
    """Tiles of 64 rows, whole tiles, CTA pairs, K slices in a cluster, a sum per plane; dense and ragged, twice in a row (the second launch behind the first)."""
    monkeypatch.setenv("DG_FORCE_BF16_FP4_FORM", "5")
    jobs = []
    for m, n, k in ((40, 264, 2048), (150, 520, 640), (600, 1032, 768), (1100, 2056, 2304)):
        codes, e, w = make_weights((n, k), 32, 210)
        jobs.append((make_rows(m, k, 211), (codes, pack_scales(e)), w, torch.empty((m, n), dtype=torch.bfloat16, device="cuda")))
    grouped = [(counts, ragged_case(counts, 2, 264, 640, 32, 212)) for counts in ([40, 0, 61, 3], [300, 64, 0, 129])]
    want = []
    for set_them in (False, True):
        for name, value in settings.items():
            if set_them:
                monkeypatch.setenv(f"DG_{name}", value)
        got = []
        for a, b, w, d in jobs:
            for _ in range(2):
                dg.bf16_fp4_gemm_nt(a, b, d.fill_(float("nan")))
            check_product(d, a, w)
            got.append(d.clone())
        for counts, (codes, e, w, a, ends) in grouped:
            d = torch.empty((a.size(0), 264), dtype=torch.bfloat16, device="cuda")
            sf = pack_scales(e)
            for _ in range(2):
                dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d.fill_(-7.0), ends)
            check_ragged(d, a, w, counts, -7.0)
            got.append(d)
        assert dg.kernel_status() == 0
        want = want or got
    assert all(torch.equal(x, y) for x, y in zip(want, got))
