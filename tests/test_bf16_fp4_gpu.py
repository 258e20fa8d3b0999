"""BF16 activations x packed E2M1 weights (bf16_fp4_gemm_nt, m_grouped_bf16_fp4_gemm_nt_ragged) against the same products in
64 bits.

Tolerance.  Per element, with S = sum |a| |w| over K:
  * the stored value is the FP32 sum rounded once: half a BF16 step, 2^-8 |value| (nothing for an FP32 D); a BF16 D that
    accumulates is read, added to and rounded again: one more 2^-8 of the larger of the two;
  * a product of a BF16 value, an E2M1 value and a power of two is exact; the sums are chains of at most K / 8 + 64
    FP32 additions (eight or more products meet in one tensor-core or FMA step), each off by at most 2^-23 of a partial
    sum that S bounds: (K / 8 + 64) 2^-23 S;
  * rows of A are split into two E4M3 values per element with one scale per 32 elements of K: what the split cannot hold is
    below 2^-14 of that scale, and the scale is at most 2^-7 of the block's largest element (amax / 448 rounded up to a power
    of two is below amax / 224): 2^-21 amax |w|, summed over K;
  * scaling by alpha: one more FP32 rounding, inside the slack of the second term.
"""
import math

import pytest
import torch

import deepgemm_amd_b200 as dg

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


@pytest.fixture(params=[0, 1, 2, 3, 4, 5], ids=["chosen", "8", "16", "16-ahead", "32-ahead", "gemm"])
def form(request, monkeypatch):
    """The ways a product is computed, each of them at every size: 8 or 16 rows a pass split inside the kernel, 16 or 32 split ahead, the GEMM kernel."""
    if request.param:
        monkeypatch.setenv("DG_FORCE_BF16_FP4_FORM", str(request.param))
    return request.param


def pack_scales(exps, mn_pad=0):
    """UE8M0 codes [G?, n, blocks] -> packed int32 [G?, n, ceil(blocks / 4)], MN-major with pitch align(n, 4) + mn_pad."""
    lead, (n, blocks) = exps.shape[:-2], exps.shape[-2:]
    pitch, words = (n + 3) // 4 * 4 + mn_pad, -(-blocks // 4)
    full = torch.zeros((*lead, words, pitch, 4), dtype=torch.uint8, device=exps.device)
    padded = torch.zeros((*lead, n, words * 4), dtype=torch.uint8, device=exps.device)
    padded[..., :blocks] = exps
    full[..., :n, :] = padded.unflatten(-1, (words, 4)).transpose(-3, -2)
    return full.view(torch.int32).squeeze(-1).transpose(-1, -2)[..., :n, :]


def make_weights(shape, gran, seed, exps=(112, 121)):
    """(codes, scale codes, W in 64 bits) for W [G?, n, k]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    *lead, n, k = shape
    codes = torch.randint(0, 256, (*lead, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    e = torch.randint(exps[0], exps[1], (*lead, n, -(-k // gran)), generator=g, device="cuda", dtype=torch.uint8)
    return codes.view(torch.int8), e, dequantise(codes, e, gran)


def dequantise(codes, e, gran):
    codes = codes.view(torch.uint8)
    k = codes.size(-1) * 2
    v = torch.tensor(E2M1, device=codes.device, dtype=torch.float64)[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    return v * torch.exp2(e.double() - 127).repeat_interleave(gran, -1)[..., :k]


def make_rows(rows, k, seed, spread=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, k), generator=g, device="cuda") * torch.exp(spread * torch.randn((rows, k), generator=g, device="cuda"))).to(torch.bfloat16)


def check_product(d, a, w, added=None, alpha=1.0):
    a, d = a.double(), d
    k = a.size(1)
    want = alpha * (a @ w.T)
    s = abs(alpha) * (a.abs() @ w.abs().T)
    amax = a.abs().unflatten(1, (k // 32, 32)).amax(-1)
    split = abs(alpha) * (amax @ w.abs().unflatten(1, (k // 32, 32)).sum(-1).T) * 2.0 ** -21
    tol = (k / 8 + 64) * 2.0 ** -23 * s + split
    if added is not None:
        want_sum = want + added.double()
        steps = want.abs().maximum(want_sum.abs())
        if d.dtype == torch.bfloat16:
            tol = tol * (1 + 2.0 ** -7) + 2.0 ** -8 * (want.abs() + want_sum.abs()) * (1 + 2.0 ** -7)
        else:
            tol = tol + 2.0 ** -23 * steps
        want = want_sum
    elif d.dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -7) + 2.0 ** -8 * want.abs()
    # below the smallest normal number of the output type the steps are absolute
    tol = tol + torch.finfo(d.dtype).smallest_normal * (2.0 ** -8 if d.dtype == torch.bfloat16 else 2.0 ** -23)
    off = (d.double() - want).abs()
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert torch.isfinite(d.float()).all() and worst <= 1.0, f"off by {worst:.3g} of the tolerance; largest difference {off.max().item():.3g}"


DENSE = [(1, 8, 128), (1, 2112, 7168), (1, 264, 16384), (2, 24, 256), (5, 100, 384), (7, 1544, 1536), (8, 40, 1152), (9, 136, 640), (15, 72, 896),
         (16, 4096, 512), (17, 48, 2048), (31, 256, 1024), (32, 80, 128), (33, 264, 2048), (61, 520, 384), (64, 576, 1152), (65, 512, 256),
         (40, 96, 256), (127, 128, 3200), (192, 1544, 256), (193, 264, 1024), (128, 2112, 512), (129, 256, 512), (300, 1000, 768), (511, 136, 128), (1030, 520, 384), (2500, 1032, 1280)]


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m,n,k", DENSE)
@pytest.mark.parametrize("gran,out", [(32, torch.bfloat16), (128, torch.float)])
def test_dense(m, n, k, gran, out):
    codes, e, w = make_weights((n, k), gran, 1000 + m)
    a = make_rows(m, k, m)
    d = torch.full((m, (n + 7) // 8 * 8), float("nan"), dtype=out, device="cuda")[:, :n]       # rows of D start on 16 bytes
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, recipe_b=(1, gran))
    check_product(d, a, w)
    again = torch.full((m, (n + 7) // 8 * 8), float("nan"), dtype=out, device="cuda")[:, :n]
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), again, recipe_b=(1, gran))
    assert torch.equal(d, again)                   # one order of summation per shape
    assert dg.kernel_status() == 0


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", [1, 6, 14, 40, 64, 150, 200, 600])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float])
@pytest.mark.parametrize("in_place", [True, False])
def test_dense_accumulates_and_scales(m, out, in_place):
    n, k = 392, 640
    codes, e, w = make_weights((n, k), 32, 3)
    a = make_rows(m, k, 4)
    c = (torch.randn((m, n), device="cuda") * 3).to(out)
    d = c.clone() if in_place else torch.full_like(c, float("nan"))
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, c=d if in_place else c, alpha=-0.37)
    check_product(d, a, w, added=c, alpha=float(torch.tensor(-0.37)))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", [1, 3, 24, 90, 400])
@pytest.mark.parametrize("gran", [32, 128])
def test_padded_pitches_and_odd_columns(m, gran):
    """Rows of every operand further apart than they are long, N odd; what lies between the rows of D stays."""
    n, k = 331, 896
    codes, e, w = make_weights((n, k), gran, 5)
    wide_w = torch.full((n, k // 2 + 64), 0x77, dtype=torch.int8, device="cuda")
    wide_w[:, : k // 2] = codes
    wide_a = torch.full((m, k + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_a[:, :k] = make_rows(m, k, 6)
    wide_d = torch.full((m, 360), -7.0, dtype=torch.bfloat16, device="cuda")
    dg.bf16_fp4_gemm_nt(wide_a[:, :k], (wide_w[:, : k // 2], pack_scales(e, mn_pad=8)), wide_d[:, :n], recipe_b=(1, gran))
    check_product(wide_d[:, :n], wide_a[:, :k], w)
    assert (wide_d[:, n:] == -7.0).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", [1, 8, 32, 70, 300])
def test_wide_ranges_of_activations_and_scales(m):
    """Rows from 2^-100 to 2^60, elements of one row 2^20 apart, rows and blocks of zeros, scale codes 0 and far apart."""
    n, k = 128, 1024
    codes, e, _ = make_weights((n, k), 32, 7, exps=(90, 150))
    e[::5, 3] = 0
    w = dequantise(codes, e, 32)
    a = make_rows(m, k, 8, spread=3.0).double()
    a *= torch.exp2(torch.linspace(-100, 60, m, device="cuda", dtype=torch.float64) if m > 1 else torch.tensor([40.0], device="cuda", dtype=torch.float64)).unsqueeze(1)
    a[:, 64:96] = 0
    if m > 2:
        a[1] = 0
    a = a.to(torch.bfloat16)
    d = torch.empty((m, n), dtype=torch.float, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
    check_product(d, a, w)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", [4, 48, 260])
def test_rows_that_are_not_finite_stay_among_themselves(m):
    n, k = 264, 512
    codes, e, w = make_weights((n, k), 32, 9)
    a = make_rows(m, k, 10)
    a[1, 37], a[2, 300] = float("inf"), float("nan")
    d = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
    assert not torch.isfinite(d[1:3].float()).any()
    keep = [0, *range(3, m)]
    check_product(d[keep], a[keep], w)


def test_fp32_scales_give_the_bits_of_packed_ones():
    for m, gran in ((3, 32), (200, 128)):
        n, k = 144, 512
        codes, e, _ = make_weights((n, k), gran, 11)
        a, d, d2 = make_rows(m, k, 12), *(torch.empty((m, n), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, recipe_b=(1, gran))
        dg.bf16_fp4_gemm_nt(a, (codes, torch.exp2(e.float() - 127)), d2, recipe_b=(1, gran))
        assert torch.equal(d, d2)


RAGGED = [([1], 0), ([0, 0, 5], 2), ([1] * 8, 0), ([3, 0, 11, 0, 0, 2, 1], 4), ([0, 17, 33, 8, 0, 64, 65, 1], 0), ([130, 0, 1, 63, 257], 7),
          ([64, 65, 128, 129, 192, 193, 1, 0, 63], 2), ([320, 64, 200, 0, 1], 0), ([0, 0, 0], 6), ([128, 256, 384], 0), ([500, 1, 2, 499], 1), ([1, 2, 3, 4] * 20, 3), ([40] * 24, 0), ([901], 0), ([0, 700, 0, 13], 5)]


def ragged_case(counts, spare, n, k, gran, seed):
    codes, e, w = make_weights((len(counts), n, k), gran, seed)
    rows = sum(counts) + spare
    a = make_rows(rows, k, seed + 1)
    ends = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    return codes, e, w, a, ends


def check_ragged(d, a, w, counts, untouched):
    start = 0
    for g, c in enumerate(counts):
        if c:
            check_product(d[start:start + c], a[start:start + c], w[g])
        start += c
    assert (d[start:] == untouched).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("counts,spare", RAGGED)
@pytest.mark.parametrize("n,k,gran", [(264, 640, 32), (1096, 1536, 128)])
def test_ragged(counts, spare, n, k, gran):
    codes, e, w, a, ends = ragged_case(counts, spare, n, k, gran, 20)
    d = torch.full((a.size(0), n), -7.0, dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends, recipe_b=(1, gran))
    check_ragged(d, a, w, counts, -7.0)
    assert dg.kernel_status() == 0


@pytest.mark.usefixtures("form")
def test_ragged_padded_pitches():
    counts, n, k = [3, 0, 70, 5], 136, 256
    codes, e, w, a, ends = ragged_case(counts, 3, n, k, 32, 30)
    wide_w = torch.full((4, n, k // 2 + 32), 0x55, dtype=torch.int8, device="cuda")
    wide_w[..., : k // 2] = codes
    for lda, ldd in ((k + 8, n + 24), (k + 64, n)):
        wide_a = torch.full((a.size(0), lda), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide_a[:, :k] = a
        wide_d = torch.full((a.size(0), ldd), -7.0, dtype=torch.bfloat16, device="cuda")
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(wide_a[:, :k], (wide_w[..., : k // 2], pack_scales(e)), wide_d[:, :n], ends)
        check_ragged(wide_d[:, :n], a, w, counts, -7.0)
        assert (wide_d[:, n:] == -7.0).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("rows", [24, 700])
def test_ragged_ends_outside_the_rows_are_clipped(rows):
    """Ends beyond the rows of A, below zero or going back make groups shorter or empty and write nothing outside D."""
    n, k = 128, 256
    codes, e, w = make_weights((5, n, k), 32, 40)
    a = make_rows(rows, k, 41)
    d = torch.full((rows, n), -7.0, dtype=torch.bfloat16, device="cuda")
    ends = torch.tensor([-3, 5, 5, rows + 100, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends)
    check_product(d[:5], a[:5], w[1])
    check_product(d[5:], a[5:], w[3])


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("rows", [40, 900])
def test_ragged_graph_replays_follow_the_ends(rows):
    n, k, groups = 264, 512, 6
    codes, e, w = make_weights((groups, n, k), 32, 50)
    sf, a = pack_scales(e), make_rows(rows, k, 51)
    ends = torch.zeros(groups, dtype=torch.int32, device="cuda")
    d = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d, ends)          # first call outside the capture: kernels are loaded
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d, ends)
    for counts in ([rows // 2, 0, 3, rows // 4, 1, 0], [0, 0, 0, 0, 0, rows], [5, 5, 5, 5, 5, 5]):
        ends.copy_(torch.tensor(counts).cumsum(0))
        a.copy_(make_rows(rows, k, 52 + counts[0]))
        d.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        check_ragged(d, a, w, counts, -7.0)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", [4, 300])
def test_two_streams_and_two_graphs_at_once(m):
    """Calls in flight together share nothing: two streams, then two graphs captured apart and replayed side by side."""
    n, k = 2112, 2048
    sides = []
    for i in range(2):
        codes, e, w = make_weights((n, k), 32, 60 + i)
        sides.append({"a": make_rows(m, k, 62 + i), "b": (codes, pack_scales(e)), "w": w, "d": torch.empty((m, n), dtype=torch.bfloat16, device="cuda"),
                      "stream": torch.cuda.Stream()})
    torch.cuda.synchronize()
    for _ in range(20):
        for s in sides:
            with torch.cuda.stream(s["stream"]):
                dg.bf16_fp4_gemm_nt(s["a"], s["b"], s["d"])
    torch.cuda.synchronize()
    for s in sides:
        check_product(s["d"], s["a"], s["w"])
        s["d"].fill_(float("nan"))
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            dg.bf16_fp4_gemm_nt(s["a"], s["b"], s["d"])
    for _ in range(20):
        for s in sides:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
    torch.cuda.synchronize()
    for s in sides:
        check_product(s["d"], s["a"], s["w"])


FORMS = [1, 14, 48, 200]                           # rows of A
RAGGED_FORMS = [3, 12, 40, 150]                    # ... of an average group


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("average", RAGGED_FORMS)
@pytest.mark.parametrize("groups", [33, 300])
def test_many_groups(groups, average):
    """More groups than a warp has lanes, sizes from zero to twice the average."""
    n, k = 264, 640
    counts = torch.randint(0, 2 * average + 1, (groups,), generator=torch.Generator().manual_seed(groups + average)).tolist()
    codes, e, w, a, ends = ragged_case(counts, 2, n, k, 32, 90)
    sf, first = pack_scales(e), None
    for _ in range(2):
        d = torch.full((a.size(0), n), -7.0, dtype=torch.bfloat16, device="cuda")
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d, ends)
        assert first is None or torch.equal(first, d)
        first = d
    check_ragged(d, a, w, counts, -7.0)
    assert dg.kernel_status() == 0


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("n,k,gran", [(4096, 2176, 128), (136, 16384, 32), (20000, 256, 32)])
@pytest.mark.parametrize("m", FORMS)
def test_slices_and_passes_of_every_form(m, n, k, gran):
    """K in slices that do not divide it, more blocks of columns than run at once, column counts that end inside a block."""
    codes, e, w = make_weights((n, k), gran, 100 + m)
    a = make_rows(m, k, 101)
    d = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, recipe_b=(1, gran))
    check_product(d, a, w)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("m", FORMS)
def test_operands_written_just_before_and_read_just_after(m, captured):
    """The kernels start before their predecessor has ended: what that one writes (weights, scales, rows) is what they read, and their results
    are complete for what follows.  Two products in a row, the second one's A and weights made from the first one's results."""
    n, k = 1024, 1024
    (c0, e0, w0), (c1, e1, w1) = make_weights((n, k), 32, 110), make_weights((k, n), 32, 111)
    sf0, sf1 = pack_scales(e0), pack_scales(e1)
    a0, a1 = make_rows(m, k, 112), make_rows(m, k, 113)
    a, codes, sf = a0.clone(), c0.clone(), sf0.clone()
    mid, out, last = (torch.empty((m, n), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    dg.bf16_fp4_gemm_nt(a, (codes, sf), mid)           # kernels loaded ahead of a capture

    def run():
        for rows, w, scales in ((a0, c0, sf0), (a1, c1, sf1)):
            a.copy_(rows)
            codes.copy_(w)
            sf.copy_(scales)
            dg.bf16_fp4_gemm_nt(a, (codes, sf), mid)
            dg.bf16_fp4_gemm_nt(mid, (codes, sf), out)
            last.copy_(out)

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    for _ in range(10):
        last.fill_(float("nan"))
        graph.replay() if captured else run()
    torch.cuda.synchronize()
    check_product(mid, a1, w1)
    check_product(last, mid, w1)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("average", RAGGED_FORMS)
def test_ends_written_just_before(average):
    groups, n, k = 40, 520, 512
    codes, e, w = make_weights((groups, n, k), 32, 120)
    sf, rows = pack_scales(e), groups * average
    a, d = make_rows(rows, k, 121), torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    ends = torch.zeros(groups, dtype=torch.int32, device="cuda")
    for seed in range(4):
        counts = torch.bincount(torch.randint(0, groups, (rows - seed,), generator=torch.Generator().manual_seed(seed)), minlength=groups)
        ready = counts.to("cuda")
        d.fill_(-7.0)
        torch.cuda.synchronize()
        for _ in range(3):
            ends.zero_()
            ends.copy_(ready.cumsum(0))
            dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d, ends)
        check_ragged(d, a, w, counts.tolist(), -7.0)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("average", RAGGED_FORMS)
def test_ragged_calls_in_flight_together(average):
    groups, n, k = 12, 1024, 768
    sides = []
    for i in range(2):
        counts = torch.randint(0, 2 * average + 1, (groups,), generator=torch.Generator().manual_seed(130 + i)).tolist()
        codes, e, w, a, ends = ragged_case(counts, 1, n, k, 32, 131 + i)
        sides.append({"args": (a, (codes, pack_scales(e)), torch.full((a.size(0), n), -7.0, dtype=torch.bfloat16, device="cuda"), ends), "w": w, "counts": counts,
                      "stream": torch.cuda.Stream()})
    torch.cuda.synchronize()
    for _ in range(20):
        for s in sides:
            with torch.cuda.stream(s["stream"]):
                dg.m_grouped_bf16_fp4_gemm_nt_ragged(*s["args"])
    torch.cuda.synchronize()
    for s in sides:
        check_ragged(s["args"][2], s["args"][0], s["w"], s["counts"], -7.0)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("m", FORMS)
def test_the_compiled_binding_and_the_ctypes_one_give_the_same_bits(m, monkeypatch):
    n, k, groups = 520, 1152, 3
    codes, e, _ = make_weights((groups, n, k), 128, 140)
    sf, a, c = pack_scales(e), make_rows(m, k, 141), torch.randn((m, n), device="cuda")
    ends = torch.tensor([m // 3, m // 3, m], dtype=torch.int32, device="cuda")
    got = []
    for binding in (dg.api._C, None):
        monkeypatch.setattr(dg.api, "_C", binding)
        for dtype in (torch.bfloat16, torch.float):
            d = torch.zeros((m, n), dtype=dtype, device="cuda")
            dg.bf16_fp4_gemm_nt(a, (codes[1], sf[1]), d, c.to(dtype), recipe_b=(1, 128), alpha=0.375)
            got.append(d)
        d = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, sf), d, ends, recipe_b=(1, 128))
        got.append(d)
    assert all(torch.equal(x, y) for x, y in zip(got[:3], got[3:]))


@pytest.mark.usefixtures("form")
def test_more_than_a_million_rows():
    m, n, k = 1_100_001, 24, 128
    codes, e, w = make_weights((n, k), 32, 150)
    a = make_rows(m, k, 151)
    d = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
    check_product(d, a, w)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("captured", [False, True])
def test_behind_a_memset_a_copy_and_a_join_of_two_streams(captured):
    """What comes before a product is not always one kernel."""
    m, n, k = 20, 1024, 768
    codes, e, w = make_weights((n, k), 32, 160)
    b, a0, host = (codes, pack_scales(e)), make_rows(m, k, 161), make_rows(m, k, 162).cpu().pin_memory()
    a, d, d2, d3 = torch.empty_like(a0), *(torch.empty((m, n), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    side = torch.cuda.Stream()
    dg.bf16_fp4_gemm_nt(a0, b, d)

    def run():
        main = torch.cuda.current_stream()
        a.copy_(host, non_blocking=True)
        dg.bf16_fp4_gemm_nt(a, b, d)                    # behind a copy from the host
        d2.zero_()
        dg.bf16_fp4_gemm_nt(a, b, d2, c=d2)             # behind a memset
        side.wait_stream(main)
        with torch.cuda.stream(side):
            a.copy_(a0)
            d3.fill_(1.0)
        d2.add_(1.0)
        main.wait_stream(side)
        dg.bf16_fp4_gemm_nt(a, b, d3, c=d3)             # behind two streams' work

    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    for _ in range(5):
        graph.replay() if captured else run()
    torch.cuda.synchronize()
    check_product(d, host.cuda(), w)
    check_product(d3, a0, w, added=torch.ones_like(d3))


@pytest.mark.usefixtures("form")
def test_the_smallest_activations():
    """Subnormal numbers and blocks below 2^-115, where the split's scale has reached its end: an element is held to 2^-21 of its block's largest, or
    to 2^-137 (2^-14 of the smallest scale, 2^-123)."""
    m, n, k = 37, 136, 512
    codes, e, w = make_weights((n, k), 32, 170, exps=(227, 236))
    g = torch.Generator(device="cuda").manual_seed(171)
    top = 0x80 * torch.randint(1, 14, (m, k // 32, 1), generator=g, device="cuda")               # blocks of subnormals up to blocks at 2^-114
    bits = (torch.rand((m, k // 32, 32), generator=g, device="cuda") * top).int() + 0x8000 * torch.randint(0, 2, (m, k // 32, 32), generator=g, device="cuda")
    a = bits.flatten(1).to(torch.int32).remainder(65536).sub(65536 * (bits.flatten(1) >= 32768)).to(torch.int16).view(torch.bfloat16)
    d = torch.empty((m, n), dtype=torch.float, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d)
    x = a.double()
    held = x.abs().unflatten(1, (k // 32, 32)).amax(-1).mul(2.0 ** -21).clamp_min(2.0 ** -137)
    tol = (k / 8 + 64) * 2.0 ** -23 * (x.abs() @ w.abs().T) + held @ w.abs().unflatten(1, (k // 32, 32)).sum(-1).T
    assert (x != 0).float().mean() > 0.9 and ((d.double() - x @ w.T).abs() <= tol).all()


def test_threads_call_at_once():
    """Host threads with products of different forms and slices, each on a stream of its own."""
    import threading
    jobs = []
    for i, (m, n, k) in enumerate([(1, 512, 4096), (6, 2112, 1024), (14, 7168, 512), (30, 1024, 2048), (90, 520, 1024), (300, 2048, 512)]):
        codes, e, w = make_weights((n, k), 32, 180 + i)
        jobs.append({"a": make_rows(m, k, 190 + i), "b": (codes, pack_scales(e)), "w": w, "d": torch.empty((m, n), dtype=torch.bfloat16, device="cuda"), "failed": None})
    for j in jobs:
        dg.bf16_fp4_gemm_nt(j["a"], j["b"], j["d"])
        j["d"].fill_(float("nan"))
    torch.cuda.synchronize()

    def work(j):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    dg.bf16_fp4_gemm_nt(j["a"], j["b"], j["d"])
                torch.cuda.current_stream().synchronize()
        except Exception as error:          # (raised in the thread: told to the test below)
            j["failed"] = error

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for j in jobs:
        assert j["failed"] is None, j["failed"]
        check_product(j["d"], j["a"], j["w"])


def test_weights_beyond_32_bit_offsets():
    """40 experts of 16384 x 8192 codes: the last ones start past 2^31 bytes."""
    groups, n, k = 40, 16384, 8192
    codes = torch.zeros((groups, n, k // 2), dtype=torch.int8, device="cuda")
    e = torch.full((groups, n, k // 32), 120, dtype=torch.uint8, device="cuda")
    last, last_e, w = make_weights((n, k), 32, 70)
    codes[-1], e[-1] = last, last_e
    a = make_rows(9, k, 71)
    ends = torch.zeros(groups, dtype=torch.int32, device="cuda")
    ends[-1] = 9
    d = torch.empty((9, n), dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (codes, pack_scales(e)), d, ends)
    check_product(d, a, w)


def test_outputs_beyond_32_bit_offsets():
    m, n, k = 70000, 32768, 128
    codes, e, w = make_weights((n, k), 128, 80)
    a = make_rows(m, k, 81)
    d = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    dg.bf16_fp4_gemm_nt(a, (codes, pack_scales(e)), d, recipe_b=(1, 128))
    for rows in (slice(0, 3), slice(65530, 65540), slice(m - 3, m)):
        check_product(d[rows], a[rows], w)
    assert dg.kernel_status() == 0


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("tokens", [1, 13, 160])
def test_an_expert_layer_end_to_end(tokens):
    """A projection, the routed rows sorted by expert, the two expert products around a gated activation, and the weighted sum
    back into the tokens: every product is checked on the inputs it was given."""
    hidden, inner, experts, top_k = 512, 384, 12, 3
    proj, proj_e, proj_w = make_weights((hidden, hidden), 128, 90)
    up, up_e, up_w = make_weights((experts, 2 * inner, hidden), 32, 91)
    down, down_e, down_w = make_weights((experts, hidden, inner), 32, 92)
    x = make_rows(tokens, hidden, 93)
    h = torch.empty_like(x)
    dg.bf16_fp4_gemm_nt(x, (proj, pack_scales(proj_e)), h, recipe_b=(1, 128))
    check_product(h, x, proj_w)
    score = torch.randn((tokens, experts), device="cuda", generator=torch.Generator(device="cuda").manual_seed(94))
    weight, expert = score.softmax(-1).topk(top_k)
    order = expert.flatten().argsort(stable=True)
    counts = torch.bincount(expert.flatten(), minlength=experts)
    ends = counts.cumsum(0).to(torch.int32)
    rows = h[order // top_k].contiguous()
    gate_up = torch.empty((rows.size(0), 2 * inner), dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(rows, (up, pack_scales(up_e)), gate_up, ends)
    check_ragged(gate_up, rows, up_w, counts.tolist(), 0)
    act = (torch.nn.functional.silu(gate_up[:, :inner].float() * 0.05) * gate_up[:, inner:].float()).to(torch.bfloat16)
    out = torch.empty((rows.size(0), hidden), dtype=torch.bfloat16, device="cuda")
    dg.m_grouped_bf16_fp4_gemm_nt_ragged(act, (down, pack_scales(down_e)), out, ends)
    check_ragged(out, act, down_w, counts.tolist(), 0)
    y = torch.zeros((tokens, hidden), device="cuda").index_add_(0, order // top_k, out.float() * weight.flatten()[order].unsqueeze(1))
    assert torch.isfinite(y).all()


def test_refusals():
    codes, e, _ = make_weights((2, 64, 256), 32, 99)
    sf, a, d = pack_scales(e), make_rows(4, 256, 1), torch.empty((4, 64), dtype=torch.bfloat16, device="cuda")
    ends = torch.tensor([1, 4], dtype=torch.int32, device="cuda")
    w0, sf0 = codes[0], pack_scales(e[0])

    def dense(a=a, w=w0, sf=sf0, d=d, **kw):
        dg.bf16_fp4_gemm_nt(a, (w, sf), d, **kw)

    def ragged(a=a, w=codes, sf=sf, d=d, ends=ends, **kw):
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (w, sf), d, ends, **kw)

    dense(), ragged()
    bad = [lambda: dense(a=a.half()), lambda: dense(a=a[:, :128]), lambda: dense(a=a[:3]), lambda: dense(a=make_rows(256, 8, 1).T[:4]),
           lambda: dense(w=w0.view(torch.uint8)), lambda: dense(w=w0.T), lambda: dense(w=w0[:, :127]), lambda: dense(sf=sf0[:32]),
           lambda: dense(sf=sf0.contiguous()), lambda: dense(d=d.half()), lambda: dense(d=d.T), lambda: dense(recipe_b=(1, 64)),
           lambda: dense(recipe_b=(1, 128)), lambda: dense(c=d.float()), lambda: dense(c=d[:, :32]), lambda: dense(w=codes, sf=sf),
           lambda: dense(a=torch.empty(4 * 260, dtype=torch.bfloat16, device="cuda")[1:4 * 256 + 1].view(4, 256)),
           lambda: dense(d=torch.empty((4, 65), dtype=torch.bfloat16, device="cuda")[:, :64]),
           lambda: dense(a=a.cpu()), lambda: dense(w=w0.cpu()), lambda: dense(sf=sf0.cpu()),
           lambda: ragged(d=d.float()), lambda: ragged(ends=ends.long()), lambda: ragged(ends=ends[:1]), lambda: ragged(ends=ends.cpu()),
           lambda: ragged(ends=ends.repeat_interleave(2)[::2]), lambda: ragged(w=codes[::2]), lambda: ragged(w=w0, sf=sf0), lambda: ragged(recipe_b=(1, 16))]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    k_small = torch.empty((4, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="k % 128 == 0"):
        dense(a=k_small, w=w0[:, :32].contiguous(), sf=pack_scales(e[0][:, :2]))


def test_empty_calls():
    codes, e, _ = make_weights((64, 256), 32, 99)
    sf = pack_scales(e)
    dg.bf16_fp4_gemm_nt(torch.empty((0, 256), dtype=torch.bfloat16, device="cuda"), (codes, sf), torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"))
    d = torch.full((3, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    empty = (torch.empty((64, 0), dtype=torch.int8, device="cuda"), torch.empty((64, 0), dtype=torch.int, device="cuda"))
    c = torch.full_like(d, 2.0)
    dg.bf16_fp4_gemm_nt(torch.empty((3, 0), dtype=torch.bfloat16, device="cuda"), empty, d, c=c)
    assert (d == 2.0).all()
    dg.bf16_fp4_gemm_nt(torch.empty((3, 0), dtype=torch.bfloat16, device="cuda"), empty, d)
    assert (d == 0.0).all() and math.isfinite(d.float().sum().item())
