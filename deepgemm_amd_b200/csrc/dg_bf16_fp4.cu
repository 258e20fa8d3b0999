// Products of BF16 activations with packed E2M1 weights and UE8M0 block scales, for a server that keeps its weights in
// four bits and its activations as they are:
//     dense    D[m, n] (+)= alpha * sum over k of A[m, k] * W[n, k]
//     ragged   D[r, n]   =          sum over k of A[r, k] * W[g(r), n, k],   group g = rows [ends[g - 1], ends[g])
//     W[n, k] = e2m1(code[n, k]) * 2^(scale code of (n, k / gran) - 127),    gran 32 or 128
// The weights and their scales lie as the FP8 x FP4 GEMMs take them (codes K-major, even K in the low nibble; scales four
// to an int32, MN-major).  An E2M1 value times a power of two times a BF16 value is exact in FP32, so the only roundings are
// those of the FP32 sums and the one of the result.
#include "dg_common.hpp"

#include <cuda_bf16.h>

#include <algorithm>

namespace dg {
namespace {

struct Bf16Fp4Params {
    const __nv_bfloat16* a;      // [m, k], pitch lda
    const uint8_t* w;            // [groups, n, k / 2], pitch ldb
    const uint32_t* sf;          // [groups][ceil(k / (4 gran))][sf_pitch]
    void* d;                     // [m, n], pitch ldd
    const int* group_ends;       // null: one group of m rows
    int m, n, k, gran;
    int64_t lda, ldb, ldd, sf_pitch;
    int accumulate;
    float alpha;
};

// Rows [first, end) of group g; ends outside [0, m] or before their predecessor give an empty group rather than a wild access
__device__ __forceinline__ void group_rows(const Bf16Fp4Params& p, int g, int& first, int& end) {
    first = 0;
    end = p.m;
    if (p.group_ends != nullptr) {
        first = g == 0 ? 0 : min(max(p.group_ends[g - 1], 0), p.m);
        end = min(max(p.group_ends[g], 0), p.m);
    }
}

// UE8M0 code -> FP32: code 0 is 2^-127 (an FP32 subnormal), code 255 has no value (infinity here, so the result shows it)
__device__ __forceinline__ float ue8m0_value(uint32_t code) { return __uint_as_float(max(code << 23, 0x00400000u)); }

__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const uint32_t e = (code >> 1) & 3, m = code & 1;
    const float size = e == 0 ? 0.5f * m : (1.0f + 0.5f * m) * static_cast<float>(1 << (e - 1));
    return code & 8 ? -size : size;
}

// One warp per column of D and up to eight rows: the lanes share K in words of eight weights, the sums meet by shuffles.
constexpr int kRowsPerPass = 8;

template <bool kDIsFP32>
__global__ void __launch_bounds__(256) bf16_fp4_kernel(const Bf16Fp4Params p) {
    const int lane = threadIdx.x % 32, n = blockIdx.x * 8 + threadIdx.x / 32, g = blockIdx.z;
    if (n >= p.n) return;
    int first, end;
    group_rows(p, g, first, end);
    const uint8_t* w = p.w + (static_cast<int64_t>(g) * p.n + n) * p.ldb;
    const int words = (p.k + 4 * p.gran - 1) / (4 * p.gran);
    const uint32_t* sf = p.sf + static_cast<int64_t>(g) * words * p.sf_pitch + n;
    for (int r0 = first + blockIdx.y * kRowsPerPass; r0 < end; r0 += gridDim.y * kRowsPerPass) {
        const int rows = min(kRowsPerPass, end - r0);
        float sum[kRowsPerPass] = {};
        for (int k0 = lane * 8; k0 < p.k; k0 += 256) {
            const uint32_t codes = *reinterpret_cast<const uint32_t*>(w + k0 / 2);
            const int block = k0 / p.gran;
            const float scale = ue8m0_value((sf[static_cast<int64_t>(block / 4) * p.sf_pitch] >> (8 * (block % 4))) & 0xFFu);
            float v[8];
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = e2m1_value((codes >> (4 * i)) & 15u);
            #pragma unroll
            for (int r = 0; r < kRowsPerPass; ++r) {
                if (r >= rows) break;
                const uint4 raw = *reinterpret_cast<const uint4*>(p.a + static_cast<int64_t>(r0 + r) * p.lda + k0);
                const uint32_t pair[4] = {raw.x, raw.y, raw.z, raw.w};
                float part = 0.0f;
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    part = fmaf(__uint_as_float(pair[i] << 16), v[2 * i], part);
                    part = fmaf(__uint_as_float(pair[i] & 0xFFFF0000u), v[2 * i + 1], part);
                }
                sum[r] = fmaf(part, scale, sum[r]);
            }
        }
        #pragma unroll
        for (int r = 0; r < kRowsPerPass; ++r) {
            if (r >= rows) break;
            #pragma unroll
            for (int off = 16; off > 0; off /= 2) sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], off);
            if (lane == 0) {
                const int64_t at = static_cast<int64_t>(r0 + r) * p.ldd + n;
                float x = sum[r] * p.alpha;
                if constexpr (kDIsFP32) {
                    float* out = static_cast<float*>(p.d) + at;
                    *out = p.accumulate ? *out + x : x;
                } else {
                    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.d) + at;
                    if (p.accumulate) x += __bfloat162float(*out);
                    *out = __float2bfloat16_rn(x);
                }
            }
        }
    }
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

    const Bf16Fp4Params p{static_cast<const __nv_bfloat16*>(g->a), static_cast<const uint8_t*>(g->b), static_cast<const uint32_t*>(g->sfb), g->d,
                          ragged ? g->grouped_layout : nullptr, g->m, g->n, g->k, g->gran_k_b, g->lda, g->ldb, g->ldd, g->sfb_pitch,
                          g->accumulate != 0, g->has_alpha ? g->alpha : 1.0f};
    const dim3 grid(ceil_div(g->n, 8), std::min(ceil_div(g->m, kRowsPerPass), ragged ? 8 : 1024), g->num_groups);
    const auto stream = static_cast<cudaStream_t>(g->stream);
    if (g->d_dtype == DG_FP32) bf16_fp4_kernel<true><<<grid, 256, 0, stream>>>(p);
    else bf16_fp4_kernel<false><<<grid, 256, 0, stream>>>(p);
    DG_CUDA_RT(cudaGetLastError());
    return DG_OK;
}

}  // namespace
}  // namespace dg

extern "C" int dg_bf16_fp4_gemm(const dg_gemm_args_t* args) { return dg::run(args, false); }
extern "C" int dg_m_grouped_bf16_fp4_gemm_ragged(const dg_gemm_args_t* args) { return dg::run(args, true); }
