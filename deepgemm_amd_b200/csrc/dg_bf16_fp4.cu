// Products of BF16 activations with packed E2M1 weights and UE8M0 block scales, for a server that keeps its weights in
// four bits and its activations as they are:
//     dense    D[m, n] (+)= alpha * sum over k of A[m, k] * W[n, k]
//     ragged   D[r, n]   =          sum over k of A[r, k] * W[g(r), n, k],   group g = rows [ends[g - 1], ends[g])
//     W[n, k] = e2m1(code[n, k]) * 2^(scale code of (n, k / gran) - 127),    gran 32 or 128
// The weights and their scales lie as the FP8 x FP4 GEMMs take them (codes K-major, even K in the low nibble; scales four
// to an int32, MN-major).  An E2M1 value times a power of two times a BF16 value is exact in FP32, so the roundings are those of the
// FP32 sums, the one of the result, and what the split of A into two E4M3 vectors cannot hold (2^-21 of the largest of 32 neighbours along K).
// A BF16 D that is added to is rounded once by the few-row kernel, which adds in FP32, and twice by the GEMM, whose TMA copy adds the rounded product: reading D in
// its epilogue instead took 500 rows, N 32768 K 512, from 29.5 us to 37.7 and 4096 rows, N 7168 K 2048, from 87 to 93.
#include "dg_common.hpp"

#include <algorithm>
#include <cmath>

#include "device/dg/bf16_fp4_few_rows.cuh"

namespace dg {

int run_split_a_gemm(const dg_gemm_args_t* args, bool ragged, int plane_rows);       // dg_gemm.cpp

namespace {

// Clusters of S CTAs that run at once with two CTAs on an SM: what 148-SM B200s showed (a cluster lives inside one GPC, and a few SMs
// belong to none that takes more than two)
int clusters_at_once(int slices) {
    static const int kFit[few::kMaxCluster + 1] = {0, 296, 148, 92, 70, 55, 44, 36, 31};
    return std::max(1, kFit[slices] * dg_get_num_sms() / 148);
}

// The few-row kernel's variants, and what a launch of each takes: so many us, and so many more for each K-block (128 x 128 weights) that a CTA
// goes through, alone on its SM or next to another one.  Fitted to 265 launches of dense products of 1 to 64 rows, N x K from 512 x 4096 to
// 7168 x 16384, in one to eight slices (4 to 95 us): half of them are met within 5 %, nine of ten within 13 %.  Ragged products, which read the
// ends before their first load, take it as it is: 8 rows in 32 groups of N 4096 K 7168 24.9 us for 25.4 measured, 131 rows of N 7168 K 2048 42.7 for 41.2, but
// 37 rows in 4 groups of N 2112 K 1536 6.4 for 8.5.  Splitting A costs a CTA
// instructions for every block (1 row 0.33 us, 8 rows 0.37); A split ahead costs a kernel more (0.8 us outside of a graph, half of it counted).
struct FewRows {
    int tokens;
    bool split;                  // splits A itself
    double fixed, alone, beside;
};
constexpr double kManyRowsLeast = 7.0;       // us that the split and the GEMM take together at least
constexpr FewRows kFewRows[] = {{8, true, 4.2, 0.23, 0.37}, {16, true, 6.0, 0.36, 0.48}, {16, false, 6.3, 0.27, 0.39}, {32, false, 7.0, 0.325, 0.45}};

// How a product is computed: a variant of the few-row kernel in so many CTAs along K (a cluster), or the GEMM kernel
struct Plan {
    const FewRows* few;          // null: the GEMM kernel on A split ahead
    int slices;
};

// Items of a launch: blocks of 128 columns of a group's rows, `tokens` of them at a time.  A ragged product's sizes are on the device: at most
// one group per row and a pass more per `tokens` rows.  Expected: no two rows in one group while there are no more rows than groups;
// above, sizes as unequal as a geometric distribution has them (c rows or more with probability q^c, q = mean / (1 + mean)), a group's passes
// being the sum of q^(1 + j tokens).
int64_t most_items(const dg_gemm_args_t* g, bool ragged, int tokens) {
    const int64_t passes = ragged ? std::min(g->m, g->num_groups + g->m / tokens) : ceil_div(g->m, tokens);
    return ceil_div(g->n, 128) * passes;
}
double expected_items(const dg_gemm_args_t* g, bool ragged, int tokens) {
    double passes = ceil_div(g->m, tokens);
    if (ragged) {
        const double q = g->m / (static_cast<double>(g->m) + g->num_groups);
        passes = g->m <= g->num_groups ? g->m : std::ceil(g->num_groups * q / (1.0 - std::pow(q, tokens)));
    }
    return ceil_div(g->n, 128) * passes;
}

Plan make_plan(const dg_gemm_args_t* g, bool ragged, int forced) {
    const int num_blocks = g->k / 128, sms = dg_get_num_sms();
    Plan best{nullptr, 0};
    double best_cost = 0.0;
    for (const FewRows& f : kFewRows) {
        if (forced >= 1 && forced <= 4 && &f != &kFewRows[forced - 1]) continue;
        const double items = expected_items(g, ragged, f.tokens);
        for (int s = 1; s <= few::kMaxCluster && (s == 1 || num_blocks / s >= 2); ++s) {
            // (CTAs that take many items do not keep step: half an item more than the average then, not a whole one)
            const double at_once = clusters_at_once(s), waves = items <= 2 * at_once ? std::ceil(items / at_once) : items / at_once + 0.5;
            const bool beside = std::min(items, at_once) * s > sms;
            // (partners finish an item before they begin the next)
            const double cost = f.fixed + waves * ceil_div(num_blocks, s) * (beside ? f.beside : f.alone) + (waves - 1) * (s > 1 ? 2.5 : 0.3);
            if (best.few == nullptr || cost < best_cost) {
                best = Plan{&f, s};
                best_cost = cost;
            }
        }
    }
    // The GEMM kernel has tiles of 64 or 128 rows of A, this one 128 columns of D and as many rows as there are: by the rows that meet one
    // matrix of weights (ragged: the average group; a pass that a group leaves half empty costs as much as a full one).  48 rows, N 4096
    // K 7168: 12.7 us, the few-row kernel 14.6; 32 rows 12.0 against 11.4; 320 rows in 16 groups 70 against 63, 400 rows 78 against 80.  Where the weights are
    // few, two launches cost more than the passes (64 rows, N 1024 K 1024: 5.7 us against 6.3).
    const int rows = ragged ? ceil_div(g->m, g->num_groups) : g->m;
    // (it stores whole 16-byte pieces of a row of D: where N ends inside one, what follows the row would not stay)
    const int d_elem = g->d_dtype == DG_FP32 ? 4 : 2;
    const bool many = forced ? forced == 5 : rows > (ragged ? 24 : 32) && best_cost > kManyRowsLeast;
    if (many && (static_cast<int64_t>(g->n) * d_elem) % 16 == 0) best = Plan{nullptr, 0};
    return best;
}

// The last sizes' plan is kept: the question is asked twice a call, and a small product takes the GPU no longer than the host
Plan plan_of(const dg_gemm_args_t* g, bool ragged) {
    struct Sizes {
        int m, n, k, groups, d_dtype, ragged, sms, forced;
        bool operator==(const Sizes& o) const {
            return m == o.m && n == o.n && k == o.k && groups == o.groups && d_dtype == o.d_dtype && ragged == o.ragged && sms == o.sms && forced == o.forced;
        }
    };
    thread_local Sizes last{};
    thread_local Plan plan{};
    // DG_FORCE_BF16_FP4_FORM: 1-4: the variants above in their order, 5: the GEMM kernel
    const Sizes now{g->m, g->n, g->k, g->num_groups, static_cast<int>(g->d_dtype), ragged, dg_get_num_sms(), env_int("FORCE_BF16_FP4_FORM")};
    if (!(now == last)) {
        plan = make_plan(g, ragged, now.forced);
        last = now;
    }
    return plan;
}

// A split ahead of the product: [hi, lo][slot][k] E4M3 bytes, then their scale words [k / 128][hi, lo][slot] (four UE8M0 codes, one per 32
// elements of K).  A dense product's slots are its rows.
struct Planes {
    uint8_t* q;
    uint32_t* sf;
    int slots;
};
int num_slots(int m, int groups, bool ragged) { return align_up(ragged ? m + 4 * groups + 4 : m, 4); }
size_t planes_bytes(int slots, int k) { return static_cast<size_t>(2) * slots * (k + k / 32); }

constexpr int kSplitRows = 16, kSplitCols = 512;

// One CTA splits 16 rows x 512 columns: 16-byte loads, quads of lanes share a scale, 8-byte stores, and the scale words of the 16 rows leave
// together (they are neighbours when the rows are).  Bound by memory: 2 bytes in, 2 + 1/16 out per element.
__global__ void __launch_bounds__(256) split_rows_kernel(const __nv_bfloat16* a, int64_t lda, const Planes out, int m, int k, const int* group_ends, int groups) {
    __shared__ int slot_of[kSplitRows];
    __shared__ uint32_t words[2][kSplitCols / 128][kSplitRows];
    // (in this order: what the product's kernel reads before it waits for this one, the weights, is then complete as well)
    griddep_wait();
    griddep_launch_dependents();
    const int row0 = blockIdx.x * kSplitRows, r = threadIdx.x / 16, chunk = threadIdx.x % 16, row = row0 + r;
    uint4 raw[kSplitCols / 128];
    #pragma unroll
    for (int b = 0; b < kSplitCols / 128; ++b) {
        const int col = blockIdx.y * kSplitCols + b * 128 + chunk * 8;
        raw[b] = make_uint4(0, 0, 0, 0);
        // (from L2: this kernel was there before its predecessor had written A, so not through the read-only path)
        if (row < m && col < k) raw[b] = __ldcg(reinterpret_cast<const uint4*>(a + row * lda + col));
    }
    // Meanwhile the first warp finds the rows' slots: a row's group is the number of ends at or before it
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, mine = row0 + lane;
        int group = 0, first = 0;
        if (group_ends != nullptr) {
            int before = 0;                                                  // the largest end of the groups ahead
            for (int g0 = 0; g0 < groups; g0 += 32) {
                int end = g0 + lane < groups ? min(max(__ldcg(group_ends + g0 + lane), 0), m) : INT32_MAX;
                const int previous = __shfl_up_sync(0xFFFFFFFFu, end, 1);
                if (__any_sync(0xFFFFFFFFu, end < (lane == 0 ? before : previous))) {      // an end that goes back is the largest so far
                    end = max(end, before);
                    #pragma unroll
                    for (int off = 1; off < 32; off *= 2) {
                        const int v = __shfl_up_sync(0xFFFFFFFFu, end, off);
                        if (lane >= off) end = max(end, v);
                    }
                }
                before = __shfl_sync(0xFFFFFFFFu, end, 31);
                #pragma unroll
                for (int i = 0; i < kSplitRows; ++i) {
                    const int behind = __popc(__ballot_sync(0xFFFFFFFFu, end <= row0 + i));
                    const int last = __shfl_sync(0xFFFFFFFFu, end, max(behind - 1, 0));
                    if (lane == i && behind > 0) {
                        group += behind;
                        first = last;
                    }
                }
            }
        }
        if (lane < kSplitRows) slot_of[lane] = mine >= m || (group_ends != nullptr && group >= groups) ? -1 : group_ends != nullptr ? first_slot(first, group) + mine - first : mine;
    }
    __syncthreads();
    const int slot = slot_of[r];
    uint2 hi[kSplitCols / 128], lo[kSplitCols / 128];
    uint32_t code[kSplitCols / 128];
    split_bf16<kSplitCols / 128>(raw, hi, lo, code);
    #pragma unroll
    for (int b = 0; b < kSplitCols / 128; ++b) {
        const int col = blockIdx.y * kSplitCols + b * 128 + chunk * 8;
        if (slot >= 0 && col < k) {
            *reinterpret_cast<uint2*>(out.q + static_cast<int64_t>(slot) * k + col) = hi[b];
            *reinterpret_cast<uint2*>(out.q + (static_cast<int64_t>(out.slots) + slot) * k + col) = lo[b];
        }
        uint32_t word = code[b] << (chunk / 4 * 8);
        word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
        word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
        if (chunk == 0) {
            words[0][b][r] = word;
            uint32_t less = 0;                                               // lo's codes: 4 less, NaN stays
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t c = word >> (8 * j) & 0xFFu;
                less |= (c == 255u ? 255u : c - 4u) << (8 * j);
            }
            words[1][b][r] = less;
        }
    }
    __syncthreads();
    if (threadIdx.x < 2 * (kSplitCols / 128) * kSplitRows) {
        const int i = threadIdx.x, rr = i % kSplitRows, b = i / kSplitRows % (kSplitCols / 128), plane = i / kSplitRows / (kSplitCols / 128);
        const int kb = blockIdx.y * (kSplitCols / 128) + b;
        if (slot_of[rr] >= 0 && kb < k / 128)
            out.sf[(static_cast<int64_t>(kb) * 2 + plane) * out.slots + slot_of[rr]] = words[plane][b][rr];
    }
}

int split_rows(const dg_gemm_args_t* g, const int* group_ends, const Planes& planes) {
    const dim3 grid(ceil_div(g->m, kSplitRows), ceil_div(g->k, kSplitCols));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(256);
    cfg.stream = static_cast<cudaStream_t>(g->stream);
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    DG_CUDA_RT(cudaLaunchKernelEx(&cfg, split_rows_kernel, static_cast<const __nv_bfloat16*>(g->a), g->lda, planes, g->m, g->k, group_ends, g->num_groups));
    return DG_OK;
}

template <int kTokens, bool kSplit>
int launch_few_rows(const dg_gemm_args_t* g, const Bf16Fp4Params& p, const Planes& planes, int slices) {
    using S = few::Shape<kTokens, kSplit>;
    const int64_t items = most_items(g, p.group_ends != nullptr, kTokens);
    CUtensorMap tm_w, tm_sf, tm_a, tm_sfa;
    int rc;
    const uint64_t words = ceil_div(g->k, 4 * g->gran_k_b);
    if ((rc = encode_tensor_map_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, g->b, g->k, static_cast<uint64_t>(g->num_groups) * g->n, g->ldb, 128, 128,
                                   CU_TENSOR_MAP_SWIZZLE_128B)) != DG_OK) return rc;
    if ((rc = encode_tensor_map_2d(&tm_sf, CU_TENSOR_MAP_DATA_TYPE_INT32, g->sfb, g->n, words * g->num_groups, g->sfb_pitch * 4, 128, 1,
                                   CU_TENSOR_MAP_SWIZZLE_NONE)) != DG_OK) return rc;
    if constexpr (kSplit) {
        if ((rc = encode_tensor_map_2d(&tm_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, g->a, g->k, g->m, g->lda * 2, 128, kTokens, CU_TENSOR_MAP_SWIZZLE_NONE)) != DG_OK) return rc;
        tm_sfa = tm_a;                           // (not used)
    } else {
        if ((rc = encode_tensor_map_2d(&tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, planes.q, g->k, static_cast<uint64_t>(2) * planes.slots, g->k, 128, kTokens,
                                       CU_TENSOR_MAP_SWIZZLE_128B)) != DG_OK) return rc;
        if ((rc = encode_tensor_map_2d(&tm_sfa, CU_TENSOR_MAP_DATA_TYPE_INT32, planes.sf, planes.slots, static_cast<uint64_t>(2) * (g->k / 128),
                                       static_cast<uint64_t>(planes.slots) * 4, kTokens, 2, CU_TENSOR_MAP_SWIZZLE_NONE)) != DG_OK) return rc;
        if ((rc = split_rows(g, p.group_ends, planes)) != DG_OK) return rc;
    }
    const auto kernel = g->gran_k_b == 32 ? few::bf16_fp4_few_rows_kernel<kTokens, kSplit, 32> : few::bf16_fp4_few_rows_kernel<kTokens, kSplit, 128>;
    const int smem = S::smem_bytes(slices);
    // (the same value every time: another thread may be between these two calls)
    static_assert(2 * (S::kMostSmem + 1024) <= 228 * 1024, "two CTAs on an SM");
    DG_CUDA_RT(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kMostSmem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(items, clusters_at_once(slices))) * slices);
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
    // Always launched behind its predecessor's start rather than its end: it waits for that kernel itself, before it reads anything that one
    // may have written, and has set up by then (2 us of a token's 6 through N 2112 K 7168)
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    DG_CUDA_RT(cudaLaunchKernelEx(&cfg, kernel, tm_w, tm_sf, tm_a, tm_sfa, p));
    return DG_OK;
}

// The GEMM kernel on the two planes (its tiles are 128 rows of A; the form above has 128 columns of D and as many rows as there are)
int launch_many_rows(const dg_gemm_args_t* g, bool ragged, const Planes& planes) {
    int rc = split_rows(g, ragged ? g->grouped_layout : nullptr, planes);
    if (rc != DG_OK) return rc;
    dg_gemm_args_t args = *g;
    args.a = planes.q;
    args.sfa = planes.sf;
    args.a_dtype = DG_FP8_E4M3;
    args.lda = g->k;
    args.gran_k_a = 32;
    args.sfa_pitch = planes.slots;
    return run_split_a_gemm(&args, ragged, planes.slots);
}

size_t workspace_bytes(const dg_gemm_args_t* g, bool ragged, const Plan& plan) {
    return plan.few != nullptr && plan.few->split ? 0 : planes_bytes(num_slots(g->m, g->num_groups, ragged), g->k);
}

int run(const dg_gemm_args_t* g, bool ragged, void* workspace, int64_t given_bytes) {
    DG_REQUIRE_ALIVE();
    DG_REQUIRE(g != nullptr);
    env_refresh();
    DG_REQUIRE(g->a_dtype == DG_BF16 && g->b_dtype == DG_FP4_E2M1_X2);
    DG_REQUIRE(g->d_dtype == DG_BF16 || (g->d_dtype == DG_FP32 && !ragged));
    DG_REQUIRE(g->major_a == DG_MAJOR_K && g->major_b == DG_MAJOR_K);
    DG_REQUIRE(g->gran_k_b == 32 || g->gran_k_b == 128);
    DG_REQUIRE(!g->stochastic_rounding && g->sfd == nullptr && g->reduce_batches <= 1 && !g->use_psum_layout);
    DG_REQUIRE(g->m >= 0 && g->n >= 0 && g->k >= 0);
    if (ragged) DG_REQUIRE(g->n > 0 && g->k > 0 && g->num_groups > 0 && g->num_groups <= 65535 && !g->accumulate && !g->has_alpha);
    else DG_REQUIRE(g->num_groups == 1);
    DG_REQUIRE(static_cast<int64_t>(g->num_groups) * g->n <= INT32_MAX);       // rows of W as a copy's coordinate
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

    const Plan plan = plan_of(g, ragged);
    const size_t needed = workspace_bytes(g, ragged, plan);
    DG_REQUIRE(needed == 0 || (workspace != nullptr && aligned(workspace, 128) && given_bytes >= 0 && static_cast<size_t>(given_bytes) >= needed));
    int rc = ensure_status_word();
    if (rc != DG_OK) return rc;
    const int slots = num_slots(g->m, g->num_groups, ragged);
    const Planes planes{static_cast<uint8_t*>(workspace), reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + static_cast<size_t>(2) * slots * g->k), slots};
    const Bf16Fp4Params p{g->d, ragged ? g->grouped_layout : nullptr, state().status_device, g->m, g->n, g->k, g->ldd, g->d_dtype == DG_FP32,
                          g->accumulate != 0, g->has_alpha ? g->alpha : 1.0f, slots, g->num_groups};
    if (plan.few == nullptr) return launch_many_rows(g, ragged, planes);
    if (plan.few->split) return plan.few->tokens == 8 ? launch_few_rows<8, true>(g, p, planes, plan.slices) : launch_few_rows<16, true>(g, p, planes, plan.slices);
    return plan.few->tokens == 16 ? launch_few_rows<16, false>(g, p, planes, plan.slices) : launch_few_rows<32, false>(g, p, planes, plan.slices);
}

}  // namespace
}  // namespace dg

extern "C" int64_t dg_bf16_fp4_workspace_bytes(const dg_gemm_args_t* args, int ragged) {
    dg::env_refresh();
    if (args == nullptr || args->m < 0 || args->n < 0 || args->k < 0 || args->num_groups <= 0) return -1;
    if (args->m == 0 || args->n == 0 || args->k == 0) return 0;
    return static_cast<int64_t>(dg::workspace_bytes(args, ragged != 0, dg::plan_of(args, ragged != 0)));
}
extern "C" int dg_bf16_fp4_gemm(const dg_gemm_args_t* args, void* workspace, int64_t workspace_bytes) { return dg::run(args, false, workspace, workspace_bytes); }
extern "C" int dg_m_grouped_bf16_fp4_gemm_ragged(const dg_gemm_args_t* args, void* workspace, int64_t workspace_bytes) {
    return dg::run(args, true, workspace, workspace_bytes);
}
