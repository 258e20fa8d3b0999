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

int run_split_a_gemm(const dg_gemm_args_t* args, bool ragged, int plane_rows);       // dg_gemm.cpp

namespace {

// Clusters of S CTAs that run at once with two CTAs on an SM: what 148-SM B200s showed (a cluster lives inside one GPC, and a few SMs
// belong to none that takes more than two)
int clusters_at_once(int slices) {
    static const int kFit[few::kMaxCluster + 1] = {0, 296, 148, 92, 70, 55, 44, 36, 31};
    return std::max(1, kFit[slices] * dg_get_num_sms() / 148);
}

// CTAs along K (a cluster) for a launch with `items` blocks of 128 columns: the number with the fewest K-blocks in a row (~0.25 us each, an
// SM's two CTAs side by side), a little more with partners, which finish an item before they begin the next
int choose_slices(int64_t items, int num_blocks) {
    int best = 1;
    double best_cost = 0.0;
    for (int s = 1; s <= few::kMaxCluster && (s == 1 || num_blocks / s >= 2); ++s) {
        const double waves = static_cast<double>(ceil_div<int64_t>(items, clusters_at_once(s)));
        const double cost = waves * (0.25 * ceil_div(num_blocks, s) + (s > 1 ? 1.5 : 0.0));
        if (s == 1 || cost < best_cost) {
            best = s;
            best_cost = cost;
        }
    }
    return best;
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
__global__ void __launch_bounds__(256) split_rows_kernel(const __nv_bfloat16* __restrict__ a, int64_t lda, const Planes out, int m, int k,
                                                         const int* __restrict__ group_ends, int groups) {
    __shared__ int slot_of[kSplitRows];
    __shared__ uint32_t words[2][kSplitCols / 128][kSplitRows];
    // (in this order: what the product's kernel reads before it waits for this one, the weights, is then complete as well)
    griddep_wait();
    griddep_launch_dependents();
    const int row0 = blockIdx.x * kSplitRows, r = threadIdx.x / 16, chunk = threadIdx.x % 16, row = row0 + r;
    if (threadIdx.x < kSplitRows) {
        const int mine = row0 + threadIdx.x;
        int slot = mine < m ? mine : -1;
        if (group_ends != nullptr && slot >= 0) {
            // the group that holds the row: the first whose end lies behind it
            int lo = 0, hi = groups;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (group_ends[mid] > mine) hi = mid;
                else lo = mid + 1;
            }
            const int first = lo == 0 ? 0 : min(max(group_ends[lo - 1], 0), m);
            slot = lo == groups ? -1 : first_slot(first, lo) + mine - first;
        }
        slot_of[threadIdx.x] = slot;
    }
    __syncthreads();
    const int slot = slot_of[r];
    uint4 raw[kSplitCols / 128];
    #pragma unroll
    for (int b = 0; b < kSplitCols / 128; ++b) {
        const int col = blockIdx.y * kSplitCols + b * 128 + chunk * 8;
        raw[b] = make_uint4(0, 0, 0, 0);
        if (slot >= 0 && col < k) raw[b] = __ldg(reinterpret_cast<const uint4*>(a + row * lda + col));
    }
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
int launch_few_rows(const dg_gemm_args_t* g, const Bf16Fp4Params& p, const Planes& planes) {
    using S = few::Shape<kTokens, kSplit>;
    // Items: exact for a dense product; a ragged one has at most one group per row, and a pass more per kTokens rows
    const int64_t tiles_n = ceil_div(g->n, 128), passes = ceil_div(g->m, kTokens);
    const int64_t items = tiles_n * (p.group_ends != nullptr ? std::min(g->m, g->num_groups + g->m / kTokens) : passes);
    const int slices = choose_slices(items, g->k / 128);
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
    DG_CUDA_RT(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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

// Which kernels a product takes, by the rows of A that meet one matrix of weights (ragged: on average; the sizes are on the device):
//   up to 8      the few-row kernel, splitting A itself; with more weights than below, and groups that hold more than 8 rows as often as not,
//                16 rows a pass on A split ahead (131 rows in 32 groups, N 7168 K 2048: 40 us against 49)
//   up to 16     the same with 16 rows a pass, as long as an SM has no more than ~16 blocks of 128 x 128 weights to go through; with more of them
//                splitting A for each costs more than a kernel that splits it once (N 7168 K 16384: 26 us against 21; N 4096 K 7168: 10.5 against 11.4)
//   up to 32     the few-row kernel on A split ahead, 32 rows a pass (ragged: up to 24, a pass that a group's size leaves half empty costs
//                as much as a full one: 320 rows in 16 groups, N 4096 K 7168: 63 us against 70 below, 400 rows 80 against 78)
//   above        the GEMM kernel on A split ahead (48 rows, N 4096 K 7168: 12.7 us, the few-row kernel in two passes 14.6; 32 rows: 12.0 against 11.4)
enum class Form { kSplit8, kSplit16, kPlanes16, kPlanes32, kMany };
Form form_of(const dg_gemm_args_t* g, bool ragged) {
    const int rows = ragged ? ceil_div(g->m, g->num_groups) : g->m;
    const int64_t blocks = static_cast<int64_t>(ceil_div(g->n, 128)) * ceil_div(g->k, 128) * (ragged ? std::min(g->num_groups, g->m) : 1);
    const bool many_blocks = blocks > static_cast<int64_t>(16) * dg_get_num_sms();
    if (rows <= 8 && !(ragged && rows > 4 && many_blocks)) return Form::kSplit8;
    if (rows <= 16) return many_blocks ? Form::kPlanes16 : Form::kSplit16;
    // (the GEMM kernel stores whole 16-byte pieces of a row of D: where N ends inside one, what follows the row would not stay)
    const int d_elem = g->d_dtype == DG_FP32 ? 4 : 2;
    return rows <= (ragged ? 24 : 32) || (static_cast<int64_t>(g->n) * d_elem) % 16 != 0 ? Form::kPlanes32 : Form::kMany;
}
bool splits_inside(const dg_gemm_args_t* g, bool ragged) {
    const Form form = form_of(g, ragged);
    return form == Form::kSplit8 || form == Form::kSplit16;
}

size_t workspace_bytes(const dg_gemm_args_t* g, bool ragged) {
    return g->m == 0 || g->n == 0 || splits_inside(g, ragged) ? 0 : planes_bytes(num_slots(g->m, g->num_groups, ragged), g->k);
}

int run(const dg_gemm_args_t* g, bool ragged, void* workspace, int64_t given_bytes) {
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

    const size_t needed = workspace_bytes(g, ragged);
    DG_REQUIRE(needed == 0 || (workspace != nullptr && aligned(workspace, 128) && given_bytes >= 0 && static_cast<size_t>(given_bytes) >= needed));
    int rc = ensure_status_word();
    if (rc != DG_OK) return rc;
    const int slots = num_slots(g->m, g->num_groups, ragged);
    const Planes planes{static_cast<uint8_t*>(workspace), reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + static_cast<size_t>(2) * slots * g->k), slots};
    const Bf16Fp4Params p{g->d, ragged ? g->grouped_layout : nullptr, state().status_device, g->m, g->n, g->k, g->ldd, g->d_dtype == DG_FP32,
                          g->accumulate != 0, g->has_alpha ? g->alpha : 1.0f, slots, g->num_groups};
    switch (form_of(g, ragged)) {
        case Form::kSplit8: return launch_few_rows<8, true>(g, p, planes);
        case Form::kSplit16: return launch_few_rows<16, true>(g, p, planes);
        case Form::kPlanes16: return launch_few_rows<16, false>(g, p, planes);
        case Form::kPlanes32: return launch_few_rows<32, false>(g, p, planes);
        case Form::kMany: break;
    }
    return launch_many_rows(g, ragged, planes);
}

}  // namespace
}  // namespace dg

extern "C" int64_t dg_bf16_fp4_workspace_bytes(const dg_gemm_args_t* args, int ragged) {
    return args == nullptr || args->m < 0 || args->k < 0 || args->num_groups <= 0 ? -1 : static_cast<int64_t>(dg::workspace_bytes(args, ragged != 0));
}
extern "C" int dg_bf16_fp4_gemm(const dg_gemm_args_t* args, void* workspace, int64_t workspace_bytes) { return dg::run(args, false, workspace, workspace_bytes); }
extern "C" int dg_m_grouped_bf16_fp4_gemm_ragged(const dg_gemm_args_t* args, void* workspace, int64_t workspace_bytes) {
    return dg::run(args, true, workspace, workspace_bytes);
}
