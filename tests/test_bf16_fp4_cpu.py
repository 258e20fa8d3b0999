"""bf16_fp4_gemm_nt and m_grouped_bf16_fp4_gemm_nt_ragged without a GPU: what the C ABI refuses before it touches the device, and
what the Python functions refuse."""
import ctypes as C

import pytest
import torch

import deepgemm_amd_b200 as dg
from deepgemm_amd_b200 import _lib


def args(**kw):
    g = _lib.GemmArgs()
    fields = dict(a=0x1000, b=0x2000, sfb=0x3000, d=0x4000, m=4, n=64, k=256, num_groups=1, a_dtype=_lib.DG_BF16, b_dtype=_lib.DG_FP4_E2M1_X2,
                  d_dtype=_lib.DG_BF16, lda=256, ldb=128, ldd=64, sfb_pitch=64, gran_k_b=32)
    for name, value in {**fields, **kw}.items():
        setattr(g, name, value)
    return g


REFUSED = [dict(a_dtype=_lib.DG_FP8_E4M3), dict(b_dtype=_lib.DG_BF16), dict(d_dtype=_lib.DG_FP8_E4M3), dict(major_a=1), dict(major_b=1),
           dict(gran_k_b=64), dict(stochastic_rounding=1), dict(sfd=0x5000), dict(reduce_batches=2), dict(use_psum_layout=1), dict(m=-1),
           dict(k=192, lda=192, ldb=96), dict(a=None), dict(b=None), dict(sfb=None), dict(d=None), dict(a=0x1008), dict(b=0x2010), dict(sfb=0x3004),
           dict(d=0x4002), dict(lda=255), dict(lda=248), dict(lda=260), dict(ldb=96), dict(ldb=144), dict(ldd=56), dict(ldd=66), dict(sfb_pitch=60),
           dict(sfb_pitch=66)]


@pytest.mark.parametrize("kw", REFUSED + [dict(num_groups=2), dict(k=0)], ids=str)
def test_dense_refuses(kw):
    assert _lib.lib.dg_bf16_fp4_gemm(C.byref(args(**kw)), None, 0) != _lib.DG_OK
    assert _lib.last_error()


@pytest.mark.parametrize("kw", REFUSED + [dict(grouped_layout=None), dict(grouped_layout=0x6002), dict(num_groups=0), dict(num_groups=65536), dict(n=0), dict(k=0),
                                          dict(accumulate=1), dict(has_alpha=1), dict(d_dtype=_lib.DG_FP32)], ids=str)
def test_ragged_refuses(kw):
    assert _lib.lib.dg_m_grouped_bf16_fp4_gemm_ragged(C.byref(args(**{"num_groups": 3, "grouped_layout": 0x6000, **kw})), None, 0) != _lib.DG_OK
    assert _lib.last_error()


def test_null_arguments_and_empty_products():
    for fn in (_lib.lib.dg_bf16_fp4_gemm, _lib.lib.dg_m_grouped_bf16_fp4_gemm_ragged):
        assert fn(None, None, 0) != _lib.DG_OK
    assert _lib.lib.dg_bf16_fp4_gemm(C.byref(args(m=0)), None, 0) == _lib.DG_OK
    assert _lib.lib.dg_bf16_fp4_gemm(C.byref(args(n=0)), None, 0) == _lib.DG_OK


def test_python_functions_refuse_cpu_tensors_and_wrong_shapes():
    a, w, sf = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros((64, 128), dtype=torch.int8), torch.zeros((2, 64), dtype=torch.int).T
    d = torch.zeros((4, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="Assertion error.*CUDA"):
        dg.bf16_fp4_gemm_nt(a, (w, sf), d)
    with pytest.raises(RuntimeError, match="m == m_"):
        dg.bf16_fp4_gemm_nt(a, (w, sf), d[:3])
    with pytest.raises(RuntimeError, match="dim"):
        dg.bf16_fp4_gemm_nt(a[0], (w, sf), d)
    with pytest.raises(RuntimeError, match="group_ends"):
        dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (w.expand(2, 64, 128).contiguous(), sf), d, torch.zeros(2, dtype=torch.int))


def test_workspace():
    size = lambda ragged=0, **kw: _lib.lib.dg_bf16_fp4_workspace_bytes(C.byref(args(**kw)), ragged)  # noqa: E731
    big = dict(n=4096, k=4096, ldb=2048, sfb_pitch=4096)
    assert size(m=8) == 0 and size(m=0) == 0 and size(m=24, num_groups=3, ragged=1) == 0 and size(m=1, **big) == 0
    assert size(m=101, **big) == 2 * 104 * (4096 + 128)                        # two planes of E4M3 and a scale per 32 of them, rows in fours
    assert size(m=101, num_groups=3, ragged=1, **big) >= 2 * (101 + 3 * 3) * (4096 + 128)        # every group starts on a multiple of four
    assert _lib.lib.dg_bf16_fp4_workspace_bytes(None, 0) == -1 and size(m=-1) == -1 and size(num_groups=0, ragged=1) == -1
    for kw in (dict(workspace=None), dict(workspace=0x7000, given=100), dict(workspace=0x7040), dict(workspace=0x7000, given=-1)):
        assert _lib.lib.dg_bf16_fp4_gemm(C.byref(args(m=64, lda=4096, ldd=4096, **big)), kw.get("workspace"), kw.get("given", 1 << 24)) != _lib.DG_OK
        assert "workspace" in _lib.last_error()


@pytest.mark.parametrize("counts", [[0, 0, 5], [1] * 8, [130, 0, 1, 63, 257], [64, 65, 128, 129, 0], [0, 0, 0], [1000]])
@pytest.mark.parametrize("ctas", [1, 7, 148])
def test_the_ragged_scheduler_visits_every_tile_of_every_group_once(counts, ctas):
    """The many-row form's walk: (first row of the tile in D, column block, group, rows that count), shared by all CTAs."""
    n, block_n = 500, 96
    ends = (C.c_int32 * len(counts))(*[sum(counts[:i + 1]) for i in range(len(counts))])
    seen = []
    for cta in range(ctas):
        out = (C.c_uint32 * 4096)()
        got = _lib.lib.dg_enumerate_tiles(_lib.DG_GEMM_M_GROUPED_RAGGED, block_n, 4, max(1, sum(counts)), n, len(counts), ends, cta, ctas, out, 1024)
        seen += [tuple(out[4 * i:4 * i + 4]) for i in range(got)]
    want = []
    for g, c in enumerate(counts):
        first = sum(counts[:g])
        for b in range(-(-c // 128)):
            want += [(first + 128 * b, j, g, min(128, c - 128 * b)) for j in range(-(-n // block_n))]
    assert sorted(seen) == sorted(want)


def test_the_many_row_configurations():
    """A stage holds 128 rows of both planes; CTA pairs for dense products of 256 rows on only; K slices only inside a cluster."""
    for m in (40, 64, 129, 300, 1024, 4096):
        for n, k in ((2112, 7168), (24576, 1536), (256, 128), (7168, 16384)):
            for kind, groups in ((_lib.DG_GEMM_DENSE, 1), (_lib.DG_GEMM_M_GROUPED_RAGGED, 8)):
                cfg = dg.get_gemm_config(kind, m, n, k, num_groups=groups, a_is_bf16=True, b_is_fp4=True, gran_k_b=32)
                assert cfg["block_m"] == 128 and cfg["block_k"] == 128 and cfg["num_stages"] >= 2 and not cfg["swap_ab"]
                assert cfg["smem_bytes"] <= 232448 and cfg["tmem_cols"] <= 512
                assert cfg["num_splits"] == 1 or cfg["split_in_cluster"]
                assert cfg["a_rows"] == (64 if m <= 64 or (groups > 1 and m <= 96 * groups) else 128)
                assert cfg["cluster_size"] == 1 or (kind == _lib.DG_GEMM_DENSE and m >= 256)
    with pytest.raises(RuntimeError):
        dg.get_gemm_config(_lib.DG_GEMM_M_GROUPED_RAGGED, 256, 512, 512, num_groups=2, b_is_fp4=True, gran_k_b=32)
    with pytest.raises(RuntimeError):
        dg.get_gemm_config(_lib.DG_GEMM_M_GROUPED_MASKED, 256, 512, 512, num_groups=2, expected_m=8, a_is_bf16=True, b_is_fp4=True, gran_k_b=32)
