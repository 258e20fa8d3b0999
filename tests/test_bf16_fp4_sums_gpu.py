"""BF16 x FP4 products, the sums: partial sums that the CTAs of a cluster exchange, and how closely FP32 sums are held."""
import pytest
import torch

import deepgemm_amd_b200 as dg
from test_bf16_fp4_gpu import check_product, check_ragged, form, make_rows, make_weights, pack_scales, ragged_case  # noqa: F401  (form: a fixture)

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


def exact_planes(m, n, k, step, seed):
    """Rows and weights of one sign whose products FP32 can add up without rounding, plane by plane, but not both planes in one sum.

    Blocks of 32 elements of K are in turn [1, 1.75] and 2^-step times that: x / s is in [256, 448] with s = 2^-8 (or 2^-(8 + step)), so hi is a multiple of 32 and
    16 times the rest, a multiple of 32 of at most 256, is lo, exactly.  Weights are 0.5 .. 6 with the scale 1.  The products of hi are multiples of
    2^-(4 + step), those of lo of 2^-(8 + step)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 1 + torch.randint(0, 97, (m, k), generator=g, device="cuda") / 128.0
    x *= torch.where(torch.arange(k, device="cuda") // 32 % 2 == 0, 1.0, 2.0 ** -step)
    codes = torch.randint(1, 8, (n, k // 2, 2), generator=g, device="cuda", dtype=torch.int32)
    w = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda", dtype=torch.float64)[codes.flatten(1)]
    packed = (codes[..., 0] | codes[..., 1] << 4).to(torch.int8)
    # the premise: hi's sum is below 2^24 of its steps, and so is lo's with all of its parts (|rest| <= 2^-4) of one sign
    hi_sum, lo_sum = (x.double() + 2.0 ** -4) @ w.T, torch.where(x >= 1, 2.0 ** -4, 2.0 ** (-4 - step)).double() @ w.T
    assert hi_sum.max() < 2.0 ** (24 - 4 - step) and lo_sum.max() < 2.0 ** (24 - 8 - step)
    return x.to(torch.bfloat16), packed, torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda"), w


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m,n,k,step,accumulate", [(1, 264, 2048, 6, False), (24, 264, 7168, 3, False), (64, 264, 7168, 3, True), (200, 264, 7168, 3, True), (200, 264, 16384, 2, True),
                                                   (1500, 1032, 7168, 3, False), (2100, 1032, 16384, 2, False), (300, 520, 2048, 6, False), (700, 520, 2048, 6, True)])
def test_sums_that_fp32_holds_are_not_cut_off(m, n, k, step, accumulate):
    """What FP32 holds of a plane's sum has to come out of it.  The roundings left are those of adding the planes (one for each slice of K, at most
    eight) and the slices (one each): 2^-24 of the result for each of 16.  (Accumulating onto zeros: one slice only, in the GEMM form.)"""
    a, codes, e, w = exact_planes(m, n, k, step, 230)
    d = torch.zeros((m, n), dtype=torch.float, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, c=d if accumulate else None)
    want = a.double() @ w.T
    assert ((d.double() - want).abs() <= 16 * 2.0 ** -24 * want).all(), ((d.double() - want) / want).abs().max().item() * 2.0 ** 24


def check_rounded(d, a, w):
    want = a.double() @ w.T
    half_step = torch.exp2(torch.floor(torch.log2(want)) - 8)
    assert ((d.double() - want).abs() <= half_step + 16 * 2.0 ** -24 * want).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m,n,k,step", [(24, 264, 7168, 3), (700, 520, 7168, 3), (2100, 1032, 16384, 2), (2100, 1032, 7168, 3)])
def test_bf16_results_are_those_sums_rounded(m, n, k, step):
    """The same sums, off by half a BF16 step and those 16 roundings: one that was cut off is on the wrong side of a border now and then."""
    a, codes, e, w = exact_planes(m, n, k, step, 231)
    d = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
    check_rounded(d, a, w)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("counts,k,step", [([9, 0, 30, 1], 7168, 3), ([300, 64, 1, 129], 7168, 3), ([700, 0, 450], 16384, 2)])
def test_ragged_results_are_those_sums_rounded(counts, k, step):
    n, ends = 520, torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    parts = [exact_planes(max(c, 1), n, k, step, 232 + i) for i, c in enumerate(counts)]
    a = torch.cat([p[0][:c] for p, c in zip(parts, counts)])
    d = torch.empty((a.size(0), n), dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (torch.stack([p[1] for p in parts]), pack_scales(torch.stack([p[2] for p in parts]))), d, ends)
    for i, (p, c) in enumerate(zip(parts, counts)):
        if c:
            check_rounded(d[int(ends[i]) - c:int(ends[i])], p[0], p[3])


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m,n,k", [(16, 520, 7168), (64, 520, 16384), (300, 520, 512), (300, 520, 1024), (600, 1032, 2048), (2100, 1032, 7168), (2100, 1032, 16384)])
def test_errors_are_those_of_a_chain_of_rounded_sums(m, n, k):
    """Against K products added in FP32 one after the other: every addition is off by at most half a step of a partial sum, 2^-24 of it, independently, and the
    partial sums of K independent terms are sqrt(i / K) of the last one, so the errors' root mean square is at most 2^-24 sqrt(K / 2) of the sums'."""
    codes, e, w = make_weights((n, k), 32, 240)
    a = make_rows(m, k, 241)
    d = torch.empty((m, n), dtype=torch.float, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
    want = a.double() @ w.T
    ratio = ((d.double() - want).pow(2).mean() / want.pow(2).mean()).sqrt().item()
    assert ratio <= 2.0 ** -24 * (k / 2) ** 0.5, ratio * 2.0 ** 24


@pytest.mark.parametrize("few", [1, 2, 3, 4])
@pytest.mark.parametrize("m,n,k", [(5, 392, 640), (30, 264, 1024), (64, 331, 640), (190, 264, 2304)])
@pytest.mark.parametrize("in_place", [True, False])
def test_few_rows_meet_a_bf16_c_in_fp32(m, n, k, in_place, few, monkeypatch):
    """C nearly cancels the product, and the one rounding is of their sum.  With S = sum |a| |w|: chains of at most K / 8 + 64 additions off by
    2^-23 S each, as for every product; the planes hold A to 2^-21 of a block's largest element; alpha and C, one FP32 rounding each of
    at most 2^-23 S; the result's, 2^-8 of it."""
    monkeypatch.setenv("DG_FORCE_BF16_FP4_FORM", str(few))
    codes, e, w = make_weights((n, k), 32, 250)
    a, alpha = make_rows(m, k, 251), -0.37
    exact = float(torch.tensor(alpha)) * (a.double() @ w.T)
    c = (exact * -(1 + 2.0 ** -6 * torch.rand(exact.shape, generator=torch.Generator(device="cuda").manual_seed(252), device="cuda"))).to(torch.bfloat16)
    wide = torch.full((m, (n + 7) // 8 * 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    d = wide[:, :n]
    if in_place:
        d.copy_(c)
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, c=d if in_place else c, alpha=alpha)
    want, s = exact + c.double(), abs(alpha) * (a.double().abs() @ w.abs().T)
    held = abs(alpha) * 2.0 ** -21 * (a.double().abs().unflatten(1, (k // 32, 32)).amax(-1) @ w.abs().unflatten(1, (k // 32, 32)).sum(-1).T)
    tol = ((k / 8 + 66) * 2.0 ** -23 * s + held) * (1 + 2.0 ** -7) + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7)
    off = (d.double() - want).abs()
    assert (off <= tol).all(), (off / tol).max().item()


@pytest.mark.parametrize("m,n,k,out", [(700, 4104, 2304, torch.bfloat16), (2300, 7176, 2304, torch.bfloat16), (200, 8200, 2304, torch.bfloat16), (700, 4104, 1152, torch.float),
                                       (200, 8204, 1152, torch.float), (3000, 2056, 640, torch.float)])
@pytest.mark.parametrize("alpha,accumulate", [(None, False), (-0.5, False), (2.0, True)])
@pytest.mark.parametrize("block_n", [0, 112, 128, 240])
def test_tiles_with_a_sum_per_plane(m, n, k, out, alpha, accumulate, block_n, monkeypatch):
    """Widths that leave tensor memory room for two tiles' sums (up to 112 columns) and for one tile's; one CTA and pairs; the last tile of 64 rows or fewer."""
    monkeypatch.setenv("DG_FORCE_BF16_FP4_FORM", "5")
    if block_n:
        monkeypatch.setenv("DG_FORCE_BLOCK_N", str(block_n))
    codes, e, w = make_weights((n, k), 32, 280)
    a, c = make_rows(m, k, 281), torch.randn((m, n), device="cuda").to(out)
    d = torch.full((m, n + 8), -7.0, dtype=out, device="cuda")[:, :n]
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, c=c if accumulate else None, alpha=alpha)
    check_product(d, a, w, added=c if accumulate else None, alpha=1.0 if alpha is None else alpha)
    assert dg.kernel_status() == 0


@pytest.mark.parametrize("block_n", [0, 112, 240])
@pytest.mark.parametrize("counts", [[300, 129, 64, 700, 0, 1], [128, 192, 20, 513], [2000, 63, 65]])
def test_ragged_tiles_with_a_sum_per_plane(counts, block_n, monkeypatch):
    monkeypatch.setenv("DG_FORCE_BF16_FP4_FORM", "5")
    if block_n:
        monkeypatch.setenv("DG_FORCE_BLOCK_N", str(block_n))
    n, k = 4104, 2304
    codes, e, w, a, ends = ragged_case(counts, 2, n, k, 32, 282)
    d = torch.full((a.size(0), n), -7.0, dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends)
    check_ragged(d, a, w, counts, -7.0)
    assert dg.kernel_status() == 0
