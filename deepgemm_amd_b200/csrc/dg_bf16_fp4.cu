// Products of BF16 activations with packed E2M1 weights and UE8M0 block scales, for a server that keeps its weights in
// four bits and its activations as they are:
//     dense    D[m, n] (+)= alpha * sum over k of A[m, k] * W[n, k]
//     ragged   D[r, n]   =          sum over k of A[r, k] * W[g(r), n, k],   group g = rows [ends[g - 1], ends[g])
//     W[n, k] = e2m1(code[n, k]) * 2^(scale code of (n, k / gran) - 127),    gran 32 or 128
// The weights and their scales lie as the FP8 x FP4 GEMMs take them (codes K-major, even K in the low nibble; scales four
// to an int32, MN-major).  An E2M1 value times a power of two times a BF16 value is exact in FP32, so the only roundings are
// those of the FP32 sums and the one of the result.
#include "dg_common.hpp"

#include <algorithm>

#include "device/dg/bf16_fp4_few_rows.cuh"

namespace dg {
namespace {

// CTAs along K (a cluster) of a launch with `tiles` CTAs of 128 columns: enough to occupy the GPU, as long as each keeps four K-blocks
int choose_slices(int64_t tiles, int ctas_per_sm, int num_blocks) {
    const int64_t slots = static_cast<int64_t>(dg_get_num_sms()) * ctas_per_sm;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({few::kMaxCluster, slots / tiles, num_blocks / 4})));
}

template <int kTokens>
int launch_few_rows(const dg_gemm_args_t* g, const Bf16Fp4Params& p) {
    using S = few::Shape<kTokens>;
    const int tiles_n = ceil_div(g->n, 128), passes = p.group_ends != nullptr ? 1 : ceil_div(g->m, kTokens);
    const int slices = choose_slices(static_cast<int64_t>(tiles_n) * passes * g->num_groups, S::kCtasPerSm, g->k / 128);
    CUtensorMap tm_w, tm_sf, tm_a;
    int rc;
    const uint64_t words = ceil_div(g->k, 4 * g->gran_k_b);
    if ((rc = encode_tensor_map_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, g->b, g->k, static_cast<uint64_t>(g->num_groups) * g->n, g->ldb, 128, 128,
                                   CU_TENSOR_MAP_SWIZZLE_128B)) != DG_OK) return rc;
    if ((rc = encode_tensor_map_2d(&tm_sf, CU_TENSOR_MAP_DATA_TYPE_INT32, g->sfb, g->n, words * g->num_groups, g->sfb_pitch * 4, 128, 1,
                                   CU_TENSOR_MAP_SWIZZLE_NONE)) != DG_OK) return rc;
    if ((rc = encode_tensor_map_2d(&tm_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, g->a, g->k, g->m, g->lda * 2, 128, kTokens, CU_TENSOR_MAP_SWIZZLE_NONE)) != DG_OK) return rc;
    const auto kernel = few::bf16_fp4_few_rows_kernel<kTokens>;
    const int smem = S::smem_bytes(slices);
    DG_CUDA_RT(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles_n * slices, passes, g->num_groups);
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(g->stream);
    cudaLaunchAttribute attrs[2];
    if (slices > 1) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[cfg.numAttrs].val.clusterDim.x = slices;
        attrs[cfg.numAttrs].val.clusterDim.y = attrs[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (state().pdl) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attrs;
    DG_CUDA_RT(cudaLaunchKernelEx(&cfg, kernel, tm_w, tm_sf, tm_a, p));
    return DG_OK;
}

int run(const dg_gemm_args_t* g, bool ragged) {
    DG_REQUIRE_ALIVE();
    DG_REQUIRE(g != nullptr);
    DG_REQUIRE(g->a_dtype == DG_BF16 && g->b_dtype == DG_FP4_E2M1_X2);
    DG_REQUIRE(g->d_dtype == DG_BF16 || (g->d_dtype == DG_FP32 && !ragged));
    DG_REQUIRE(g->major_a == DG_MAJOR_K && g->major_b == DG_MAJOR_K);
    DG_REQUIRE(g->gran_k_b == 32 || g->gran_k_b == 128);
    DG_REQUIRE(!g->stochastic_rounding && g->sfd == nullptr && g->reduce_batches <= 1 && !g->use_psum_layout);
    DG_REQUIRE(g->m >= 0 && g->n >= 0 && g->k >= 0);
    if (ragged) DG_REQUIRE(g->n > 0 && g->k > 0 && g->num_groups > 0 && g->num_groups <= 65535 && !g->accumulate && !g->has_alpha);
    else DG_REQUIRE(g->num_groups == 1);
    if (g->m == 0 || g->n == 0) return DG_OK;
    if (g->k == 0) return fail(DG_ERR_INVALID_ARGUMENT, "k == 0 must be handled by the caller (zero or copy D)");
    DG_REQUIRE(g->k % 128 == 0);                                           // as for every packed FP4 operand
    DG_REQUIRE(g->a != nullptr && g->b != nullptr && g->sfb != nullptr && g->d != nullptr && (!ragged || g->grouped_layout != nullptr));
    const auto aligned = [](const void* ptr, uintptr_t al) { return reinterpret_cast<uintptr_t>(ptr) % al == 0; };
    DG_REQUIRE(aligned(g->a, 16) && aligned(g->b, 32) && aligned(g->sfb, 16) && aligned(g->d, 16) && aligned(g->grouped_layout, 4));
    DG_REQUIRE(g->lda >= g->k && g->lda % 8 == 0);
    DG_REQUIRE(g->ldb >= g->k / 2 && g->ldb % 32 == 0);
    const int d_elem = g->d_dtype == DG_FP32 ? 4 : 2;
    DG_REQUIRE(g->ldd >= g->n && (g->ldd * d_elem) % 16 == 0);
    DG_REQUIRE(g->sfb_pitch >= align_up<int64_t>(g->n, 4) && g->sfb_pitch % 4 == 0);

    int rc = ensure_status_word();
    if (rc != DG_OK) return rc;
    const Bf16Fp4Params p{g->d, ragged ? g->grouped_layout : nullptr, state().status_device, g->m, g->n, g->k, g->gran_k_b,
                          g->ldd, g->d_dtype == DG_FP32, g->accumulate != 0, g->has_alpha ? g->alpha : 1.0f};
    const int rows = ragged ? ceil_div(g->m, g->num_groups) : g->m;
    if (rows <= 8) return launch_few_rows<8>(g, p);
    if (rows <= 16) return launch_few_rows<16>(g, p);
    if (rows <= 32) return launch_few_rows<32>(g, p);
    return launch_few_rows<64>(g, p);
}

}  // namespace
}  // namespace dg

extern "C" int dg_bf16_fp4_gemm(const dg_gemm_args_t* args) { return dg::run(args, false); }
extern "C" int dg_m_grouped_bf16_fp4_gemm_ragged(const dg_gemm_args_t* args) { return dg::run(args, true); }
