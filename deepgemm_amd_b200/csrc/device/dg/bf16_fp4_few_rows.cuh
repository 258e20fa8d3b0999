// D = A W^T for a few BF16 rows of A and packed E2M1 weights W with UE8M0 block scales: the decode form of the BF16 x FP4
// products.  What bounds it is the bytes of W, half a byte per weight, as long as nothing has to touch every weight: a token through
// N 7168 K 16384 takes 14.9 us, 62 MB of weights and scales, of which ~4 us are the launch, the first stage and the cluster's exchange.
//
// Mathematics.  The tensor cores multiply E2M1 by E4M3 with a power-of-two scale per 32 elements of K on either side
// (tcgen05.mma.kind::mxf8f6f4), so W goes in as it is.  A BF16 value has 8 significant bits and an E4M3 value 4: every 32 elements
// of a row of A become two E4M3 vectors with scales s and s / 16,
//     x = s hi + (s / 16) lo,     hi = e4m3(x / s),  lo = e4m3(16 (x / s - hi)),
// s being the smallest power of two with |x| / s <= 448.  hi leaves a remainder of at most half its last place, which is a multiple of
// x's own last place: at most 8 of them, so four bits hold it and the split is exact, down to |x| = 2^-6 s; below that it
// is off by at most 2^-14 s <= 2^-21 of the block's largest element.  A row of A is thus two columns of the tile, `hi` and `lo`,
// whose FP32 accumulators are added at the end.  (Unpacking W to FP16 for the register-operand MMA instead costs
// some 28 instructions per 512 weights, which held a kernel built that way to 3.3 TB/s of W; here no instruction is spent on W.)
//
// Work.  W is the 128-row operand: an item is 128 columns of D times up to kTokens rows of A (2 kTokens tile columns).  CTAs stay and take
// items in turn; the accumulators are double, so an item's epilogue runs under the next one's loads and products.
//   warp 0      TMA producer: per 128 elements of K 128 rows of W (8 KB, unpacked to a byte each on the way), their scale words, and A
//   warps 1, 3  MMA issuers (narrow tiles: both, taking K-blocks in turn; their accumulators are added at the end)
//   warp 2      allocates tensor memory, rearranges scale words for tcgen05.cp
//   warps 4-7   epilogue
//   warps 8-15  in teams of two: split a stage's rows of A into its tile columns and their scales.  For more rows, or more weights to a
// CTA, splitting them again in every CTA costs more than the weights (a block of 16 rows takes a CTA 0.36 us instead of 0.27): a kernel of its own
// then does it once and this one, without those warps, loads the two planes; it asks for the first stages of W before that kernel is done.
// Where the items alone do not occupy the GPU, the CTAs of a cluster (up to 8) share an item's K and send their partial sums to one another
// through distributed shared memory, every CTA adding up its own rows of D in rank order.  A block of 8 KB takes a CTA 0.23 us where it has its
// SM to itself (the issuing warps' walks around their loops) and 0.37 next to another one, as fitted over launches of 1 to 64 rows; a token's 62 MB
// through N 7168 K 16384 (224 CTAs, two to an SM on 76 of them) arrive at 5.6 TB/s between the launch's start and its end, a copy's rate being 6.56.  Asking L2 for
// weights further ahead than the ring of stages cost 3 to 20 %.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ptx.cuh"
#include "tile_scheduler.cuh"

namespace dg {

struct Bf16Fp4Params {
    void* d;                     // [m, n], pitch ldd
    const int* group_ends;       // null: one group of m rows
    int* status;                 // host-visible status word, 0 = ok
    int m, n, k;
    int64_t ldd;
    int d_fp32, accumulate;
    float alpha;
    int slots;                   // A split ahead: slots per plane (hi, then lo)
    int groups;
};

// One thread's share of the split: N pieces of eight elements of a row, the four threads of an aligned quad holding 32 consecutive ones.
// hi, lo: eight E4M3 values each; code: UE8M0 code of hi's scale (lo's is 4 less), 255 (NaN) for a block with an infinity or NaN.
template <int N>
__device__ __forceinline__ void split_bf16(const uint4 (&raw)[N], uint2 (&hi)[N], uint2 (&lo)[N], uint32_t (&code)[N]) {
    uint32_t most[N];
    #pragma unroll
    for (int p = 0; p < N; ++p) {
        const uint4& x = raw[p];
        const uint32_t most2 = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
        most[p] = max(most2 & 0xFFFFu, most2 >> 16);                         // the bits of |x| order like |x|
    }
    #pragma unroll
    for (int p = 0; p < N; ++p) most[p] = max(most[p], __shfl_xor_sync(0xFFFFFFFFu, most[p], 1));
    #pragma unroll
    for (int p = 0; p < N; ++p) most[p] = max(most[p], __shfl_xor_sync(0xFFFFFFFFu, most[p], 2));
    #pragma unroll
    for (int p = 0; p < N; ++p) {
        const uint32_t x[4] = {raw[p].x, raw[p].y, raw[p].z, raw[p].w};
        // |x| = f 2^e with 448 = 1.75 2^8: the code of s is e - 8, one more when f > 1.75.  (Not below 4, so that lo has a code: a block
        // whose largest element is below 2^-115 is then held to 2^-137)
        const uint32_t c = max(static_cast<int>((most[p] >> 7) + ((most[p] & 0x7Fu) > 0x60u ? 1u : 0u)) - 8, 4);
        const __nv_bfloat16 inv = __ushort_as_bfloat16(static_cast<unsigned short>((254u - c) << 7));      // 1 / s
        uint32_t h[4], l[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]), __halves2bfloat162(inv, inv));  // exact
            const uint32_t bits = *reinterpret_cast<const uint32_t*>(&y);
            const __half2 f = __floats2half2_rn(__uint_as_float(bits << 16), __uint_as_float(bits & 0xFFFF0000u));           // |y| <= 448: exact from 2^-17 on
            uint16_t q;
            uint32_t back;
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(q) : "r"(*reinterpret_cast<const uint32_t*>(&f)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(q));
            const __half2 rest = __hmul2(__hsub2(f, *reinterpret_cast<const __half2*>(&back)), __float2half2_rn(16.0f));
            uint16_t r;
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
            h[i] = q;
            l[i] = r;
        }
        hi[p] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        lo[p] = make_uint2(l[0] | (l[1] << 16), l[2] | (l[3] << 16));
        code[p] = most[p] >= 0x7F80u ? 255u : c;
    }
}

namespace few {

constexpr uint32_t kRoleSplit = 8;           // role code of the splitting warps' waits (status word); the others are the GEMM kernel's
constexpr int kMaxCluster = 8;

// A bounded wait whose outcome the whole warp shares (some lanes may see the barrier complete just as others give up)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const AbortCtx& ctx, uint32_t role) {
    const bool ok = mbar_wait(bar, parity, ctx, role, 1);
    return __all_sync(0xFFFFFFFFu, ok) != 0;
}

// One thread of the warp, the same one every time
__device__ __forceinline__ bool elect_one() {
    uint32_t elected;
    asm volatile("{.reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.b32 %0, 1, 0, p;}" : "=r"(elected));
    return elected != 0;
}
// A value that lane `l` holds, to all lanes.  (A reduction rather than a shuffle: its result is known to be the same in the whole warp, so what
// is computed from it, the MMA's descriptors above all, stays in uniform registers)
__device__ __forceinline__ int from_lane(int v, int l) { return __reduce_add_sync(0xFFFFFFFFu, static_cast<int>(lane_id()) == l ? v : 0); }

// The items in their order: groups, in a group its blocks of 128 columns, for each of them the passes of kTokens rows.  Lane l of a warp
// holds group `window + l`, so finding an item takes a ballot, and 32 groups are passed over with one load.
template <int tokens>
struct Items {
    int groups, tiles, window = -32, before = 0;              // items of the groups ahead of the window
    int window_first = 0;                                     // where the groups ahead of the window end
    int my_first = 0, my_rows = 0, my_end = 0;                // this lane's group: its rows, the items up to and with it
    int group, first, rows, row, n0;                          // the item: its group, that one's rows, first row of the pass, first column

    __device__ explicit Items(const Bf16Fp4Params& p) : groups(p.groups), tiles((p.n + 127) / 128) {
        group = first = row = 0;
        rows = p.m;
    }

    // The warp together; items in growing order
    __device__ __forceinline__ bool find(const Bf16Fp4Params& p, int item) {
        if (p.group_ends == nullptr) {                        // one group: no search
            const int passes = (rows + tokens - 1) / tokens, tile = passes == 1 ? item : item / passes;
            row = (item - tile * passes) * tokens;
            n0 = tile * 128;
            return tile < tiles;
        }
        int end = window < 0 ? 0 : from_lane(my_end, 31);
        while (item >= end) {
            if (window + 32 >= groups) return false;
            window += 32;
            before = end;
            const int g = window + static_cast<int>(lane_id());
            // A group begins where the one before it ends; an end outside [0, m] is moved to its border, one before an earlier end is that one.
            // (From L2: with A split ahead they are read before the kernel before this one is done)
            int last = g < groups ? min(max(__ldcg(p.group_ends + g), 0), p.m) : p.m;
            auto previous = [&]() {
                const int v = __shfl_up_sync(0xFFFFFFFFu, last, 1);
                return lane_id() == 0 ? window_first : v;
            };
            my_first = previous();
            if (__any_sync(0xFFFFFFFFu, last < my_first)) {   // ends that go back: the largest so far
                last = max(last, window_first);
                #pragma unroll
                for (int off = 1; off < 32; off *= 2) {
                    const int v = __shfl_up_sync(0xFFFFFFFFu, last, off);
                    if (static_cast<int>(lane_id()) >= off) last = max(last, v);
                }
                my_first = previous();
            }
            window_first = from_lane(last, 31);
            my_rows = g < groups ? last - my_first : 0;
            my_end = tiles * ((my_rows + tokens - 1) / tokens);
            #pragma unroll
            for (int off = 1; off < 32; off *= 2) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, my_end, off);
                if (static_cast<int>(lane_id()) >= off) my_end += v;
            }
            my_end += before;
            end = from_lane(my_end, 31);
        }
        const int l = __ffs(__ballot_sync(0xFFFFFFFFu, item < my_end)) - 1;
        group = window + l;
        first = from_lane(my_first, l);
        rows = from_lane(my_rows, l);
        const int passes = (rows + tokens - 1) / tokens, local = item - (from_lane(my_end, l) - tiles * passes);
        const int tile = passes == 1 ? local : local / passes;
        row = first + (local - tile * passes) * tokens;
        n0 = tile * 128;
        return true;
    }
    __device__ __forceinline__ int rows_here() const { return min(tokens, first + rows - row); }
};

// kSplit: the kernel splits A itself; otherwise A comes as the two planes of a kernel before this one
template <int kTokens, bool kSplit> struct Shape {
    static constexpr int kCols = 2 * kTokens;                                // columns of the tile
    static constexpr int kStages = kTokens == 8 ? 5 : (kTokens == 16 ? 4 : 3);      // two CTAs share an SM's 227 KB
    // Teams of splitting warps take turns at the K-blocks: a block's chain of wait, shuffles, conversions, stores and fence is long, so as
    // many blocks as possible are at it at once
    static constexpr int kTeams = 4, kTeam = 2, kPieces = kTokens / (2 * kTeam), kSplitWarps = kTeams * kTeam;
    static constexpr int kThreads = kSplit ? 256 + 32 * kSplitWarps : 256;
    static_assert(!kSplit || (kTokens <= 16 && kTeams <= kStages), "a team that is done with its last block knows that the stage of its next one is at most one block behind");
    static constexpr int kOffB = kStages * 16384, kOffA = kOffB + kStages * kCols * 128, kOffSfa = kOffA + (kSplit ? kStages * kTokens * 256 : 0), kOffSfb = kOffSfa + kStages * 512;
    static constexpr int kOffBar = kOffSfb + kStages * 512, kOffMisc = kOffBar + (4 * kStages + 4) * 8, kOffRecv = (kOffMisc + 8 + 15) / 16 * 16;
    // MMA-issuing warps, taking K-blocks in turn: with tiles this narrow a warp's walk around its loop takes 550 cycles, the MMAs 100.  Each
    // has accumulators and scale columns of its own (what two threads issue has no order).  (7 rows, N 24576 K 1536: 8.6 -> 8.2 us; 131 rows in
    // 32 groups of N 7168 K 2048, 8 a pass: 43 -> 40.  16 rows split inside are bound by the splitting, 32 by the MMAs)
    static constexpr int kIssuers = kTokens * (kSplit ? 2 : 1) <= 16 ? 2 : 1;
    static constexpr int kScaleCol = 2 * kIssuers * kCols, kTmemUsed = kScaleCol + 8 * kIssuers;
    static constexpr int kTmemCols = kTmemUsed <= 64 ? 64 : (kTmemUsed <= 128 ? 128 : 256);
    static_assert(kTokens <= 32, "two CTAs' shares of an SM's shared and tensor memory");
    // What a CTA receives: every slice's partial sums of the rows of D it owns
    __host__ __device__ static constexpr int recv_rows(int slices) { return (kTokens + slices - 1) / slices; }
    static constexpr int kMostSmem = kOffRecv + (kTokens + kMaxCluster - 1) * 512;
    __host__ __device__ static constexpr int smem_bytes(int slices) { return kOffRecv + (slices > 1 ? slices * recv_rows(slices) * 512 : 0); }
};

// kGran: elements of K per scale of W
template <int kTokens, bool kSplit, int kGran>
__global__ void __launch_bounds__(Shape<kTokens, kSplit>::kThreads, 2)
bf16_fp4_few_rows_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_sf, const __grid_constant__ CUtensorMap tm_a,
                         const __grid_constant__ CUtensorMap tm_sfa, const Bf16Fp4Params p) {
    using S = Shape<kTokens, kSplit>;
    constexpr uint32_t kStages = S::kStages, kCols = S::kCols;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t warp = __reduce_max_sync(0xFFFFFFFFu, threadIdx.x / 32), lane = lane_id();
    const uint32_t base = smem_u32(smem);
    auto full_bar = [&](uint32_t s) { return base + S::kOffBar + s * 8; };
    auto sf_bar = [&](uint32_t s) { return base + S::kOffBar + (kStages + s) * 8; };
    auto empty_bar = [&](uint32_t s) { return base + S::kOffBar + (2 * kStages + s) * 8; };
    auto a_bar = [&](uint32_t s) { return base + S::kOffBar + (3 * kStages + s) * 8; };
    auto done_bar = [&](uint32_t a) { return base + S::kOffBar + (4 * kStages + a) * 8; };
    auto free_bar = [&](uint32_t a) { return base + S::kOffBar + (4 * kStages + 2 + a) * 8; };
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::kOffMisc);
    volatile uint32_t* const abort_flag = tmem_slot + 1;
    const AbortCtx ctx{abort_flag, p.status};
    uint32_t slices;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(slices));
    const uint32_t rank = cluster_ctarank();

    const int num_blocks = p.k / 128, per_slice = (num_blocks + slices - 1) / slices;
    const int kb0 = min(static_cast<int>(rank) * per_slice, num_blocks), kb1 = min(kb0 + per_slice, num_blocks);
    const bool some = kb1 > kb0;                 // (a slice beyond the end of K has nothing to add)
    const int step = gridDim.x / slices, first_item = blockIdx.x / slices;
    Items<kTokens> at(p);
    uint32_t stage = 0, phase = 0;
    auto advance = [&]() {
        stage = stage + 1 == kStages ? 0 : stage + 1;
        phase ^= stage == 0;
    };
    // The copies of K-block kb of the item into the current stage (one thread)
    auto load_w = [&](int kb) {
        mbar_arrive_expect_tx(sf_bar(stage), 512 + (kSplit ? 0 : kCols * 4));
        tma_load_2d(base + S::kOffSfa + stage * 512, &tm_sf, sf_bar(stage), at.n0, at.group * ((p.k + 4 * kGran - 1) / (4 * kGran)) + (kGran == 32 ? kb : kb / 4));
        mbar_arrive_expect_tx(full_bar(stage), 128 * 64 + (kSplit ? 0 : kCols * 128));
        tma_load_2d(base + stage * 16384, &tm_w, full_bar(stage), kb * 128, at.group * p.n + at.n0);
    };
    auto load_a = [&](int kb) {
        if constexpr (kSplit) {
            mbar_arrive_expect_tx(a_bar(stage), kTokens * 256);
            tma_load_2d(base + S::kOffA + stage * kTokens * 256, &tm_a, a_bar(stage), kb * 128, at.row);
        } else {
            const int slot = (p.group_ends != nullptr ? first_slot(at.first, at.group) : 0) + at.row - at.first;
            tma_load_2d(base + S::kOffSfb + stage * 512, &tm_sfa, sf_bar(stage), slot, 2 * kb);      // hi's words, then lo's
            #pragma unroll
            for (int plane = 0; plane < 2; ++plane)
                tma_load_2d(base + S::kOffB + stage * kCols * 128 + plane * kTokens * 128, &tm_a, full_bar(stage), kb * 128, plane * p.slots + slot);
        }
    };

    // The producer asks for the first item's first stages (all of them free) while the others still set up.  With A split ahead, what the
    // kernel before this one wrote is A alone, so W is asked for before that kernel is waited for (it was itself launched behind everything
    // that came before); A follows below.
    int ahead = kb0;                             // K-blocks of the first item asked for here
    if (warp == 0) {
        if (lane == 0) {
            *abort_flag = 0;
            for (uint32_t s = 0; s < kStages; ++s) {
                mbar_init(full_bar(s), 2 + (kSplit ? S::kTeam : 0));       // the producer, the rearranging warp, a team of splitting warps
                mbar_init(sf_bar(s), 1);
                mbar_init(empty_bar(s), 1);      // tcgen05.commit
                mbar_init(a_bar(s), 1);
            }
            for (uint32_t a = 0; a < 2; ++a) {
                mbar_init(done_bar(a), S::kIssuers);       // tcgen05.commit: an item's accumulators are complete
                mbar_init(free_bar(a), 4);       // the epilogue warps have read them
            }
            fence_mbar_init();
        }
    } else if (warp == 2) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_slot)), S::kTmemCols);
        tmem_relinquish<1>();
    }
    __syncwarp();
    // (every warp by itself, here: a ragged product's first item takes ~1 us to find)
    if (kSplit) griddep_wait();
    bool found = at.find(p, first_item);
    if (warp == 0) {
        if (found) {
            ahead = min(kb0 + static_cast<int>(kStages), kb1);
            for (int kb = kb0; kb < ahead; ++kb, ++stage) {
                if (elect_one()) {
                    if (kSplit) load_a(kb);
                    load_w(kb);
                }
            }
            stage = 0;
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __reduce_max_sync(0xFFFFFFFFu, *tmem_slot);
    auto accumulators = [&](uint32_t a, uint32_t issuer) { return tmem + (a * S::kIssuers + issuer) * kCols; };
    griddep_wait();
    griddep_launch_dependents();
    bool ok = true;

    // Every warp walks the same items and K-blocks
    uint32_t count = 0, steps = 0;               // items so far: accumulator count % 2; their K-blocks (splitting warps)
    for (int item = first_item; found; item += step, found = at.find(p, item), ++count) {
        const uint32_t accum = count & 1, accum_phase = count >> 1 & 1;
        // first half of a split barrier: this CTA runs, and what it received for the item before has been read (so a release from the
        // second item on: those reads come before what the peers write there next)
        if (slices > 1) {
            if (count == 0) cluster_arrive_relaxed();
            else cluster_arrive();
        }
        if (warp == 0) {
            int kb = kb0;
            if (count == 0) {
                for (; kb < ahead; ++kb, advance())
                    if (!kSplit && elect_one()) load_a(kb);
                __syncwarp();
            }
            for (; ok && kb < kb1; ++kb, advance()) {
                if (!(ok = warp_wait(empty_bar(stage), phase ^ 1, ctx, 1))) break;
                if (elect_one()) {
                    load_a(kb);
                    load_w(kb);
                }
                __syncwarp();
            }
        } else if (warp == 1 || (S::kIssuers == 2 && warp == 3)) {
            constexpr uint32_t idesc = make_instr_desc_block_scaled(kFmtE2M1, kFmtE4M3, 0, 0, 128, kCols);
            const int me = warp == 1 ? 0 : 1, blocks = kb1 - kb0;
            const uint32_t tmem_d = accumulators(accum, me), tmem_sfa = tmem + S::kScaleCol + 8 * me, tmem_sfb = tmem_sfa + 4;
            if (some) ok = ok && warp_wait(free_bar(accum), accum_phase ^ 1, ctx, 2);
            tc_fence_after_sync();
            if (some && me >= blocks && lane == 0) mbar_arrive(done_bar(accum));       // (nothing to do for the second one)
            for (int b = 0; ok && b < blocks; ++b, advance()) {
                if (b % S::kIssuers != me) continue;
                // First that the stage's block before this one, perhaps the other warp's, has been multiplied (a barrier two phases behind answers
                // like one that is done)
                if (S::kIssuers > 1 && !(ok = warp_wait(empty_bar(stage), phase ^ 1, ctx, 2))) break;
                if (!(ok = warp_wait(full_bar(stage), phase, ctx, 2))) break;
                tc_fence_after_sync();
                const int kb = kb0 + b;
                const uint64_t a_desc = make_smem_desc(base + stage * 16384, 0, 1024, kSwizzle128B);
                const uint64_t b_desc = make_smem_desc(base + S::kOffB + stage * kCols * 128, 0, 1024, kSwizzle128B);
                const uint64_t sfa_desc = make_smem_desc(base + S::kOffSfa + stage * 512, 0, 128, kSwizzleNone);
                const uint64_t sfb_desc = make_smem_desc(base + S::kOffSfb + stage * 512, 0, 128, kSwizzleNone);
                if (elect_one()) {
                    tc_cp_32x128b_warpx4<1>(tmem_sfa, sfa_desc);
                    tc_cp_32x128b_warpx4<1>(tmem_sfb, sfb_desc);
                    #pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        tc_mma_mxf8f6f4<1>(tmem_d, a_desc + j * 2, b_desc + j * 2, instr_desc_with_sf_ids(idesc, kGran == 32 ? j : kb % 4, j),
                                           tmem_sfa, tmem_sfb, b != me || j != 0);
                    tc_commit(empty_bar(stage));
                    if (b + S::kIssuers >= blocks) tc_commit(done_bar(accum));
                }
                __syncwarp();
            }
        } else if (warp == 2) {
            // tcgen05.cp puts row r of 32 x 16 bytes into lane r: the word of tile row 32 c + r has to sit at word 4 r + c
            for (int kb = kb0; ok && kb < kb1; ++kb, advance()) {
                if (!(ok = warp_wait(sf_bar(stage), phase, ctx, 3))) break;
                const uint32_t words = base + S::kOffSfa + stage * 512, own = base + S::kOffSfb + stage * 512;
                uint32_t v[4], w[4];
                #pragma unroll
                for (uint32_t c = 0; c < 4; ++c) v[c] = ld_shared_u32(words + (c * 32 + lane) * 4);
                if constexpr (!kSplit) {                                     // the same for the scale words of A (the splitting warps write theirs in place)
                    #pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) w[c] = c * 32 < kCols ? ld_shared_u32(own + (c * 32 + lane) * 4) : 0u;
                }
                __syncwarp();
                st_shared_v4(words + lane * 16, v[0], v[1], v[2], v[3]);
                if constexpr (!kSplit) st_shared_v4(own + lane * 16, w[0], w[1], w[2], w[3]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(stage));
                __syncwarp();
            }
        } else if (warp >= 8) {
            const int rows = at.rows_here(), blocks = kb1 - kb0, team = (warp - 8) / S::kTeam, member = (warp - 8) % S::kTeam;
            // Piece i of this lane: elements 8 (lane % 16) .. of the K-block, of row 2 (i kTeam + member) + lane / 16.  (stage, phase: those of
            // the item's first block)
            const int row0 = member * 2 + lane / 16, chunk = lane % 16;
            uint32_t b_stage = stage, b_phase = phase;
            for (int b = 0; ok && b < blocks; ++b) {
                const uint32_t at_stage = b_stage, at_phase = b_phase;
                b_stage = b_stage + 1 == kStages ? 0 : b_stage + 1;
                b_phase ^= b_stage == 0;
                // (counted over all items: a team is then never more than kTeams blocks away from its last one)
                if ((steps + b) % S::kTeams != static_cast<uint32_t>(team)) continue;
                // First that the stage's block before this one has been multiplied, then that this one's A has landed.  Copies land in any
                // order, and a warp that only asked for the latter could ask while the copy of the block before is still
                // under way: a barrier two phases behind answers like one that is done.
                if (!(ok = warp_wait(empty_bar(at_stage), at_phase ^ 1, ctx, kRoleSplit))) break;
                if (!(ok = warp_wait(a_bar(at_stage), at_phase, ctx, kRoleSplit))) break;
                const uint8_t* const a = smem + S::kOffA + at_stage * kTokens * 256 + chunk * 16;
                uint8_t* const tile = smem + S::kOffB + at_stage * kCols * 128;
                uint8_t* const sf = smem + S::kOffSfb + at_stage * 512;
                // (pieces side by side, so that their chains of shuffles and conversions overlap; rows beyond the last one are split along with
                // the others: their columns are not stored)
                auto split = [&](auto pieces) {
                    constexpr int kN = decltype(pieces)::value;
                    uint4 raw[kN];
                    uint2 hi[kN], lo[kN];
                    uint32_t code[kN];
                    #pragma unroll
                    for (int i = 0; i < kN; ++i) raw[i] = *reinterpret_cast<const uint4*>(a + (row0 + 2 * S::kTeam * i) * 256);
                    split_bf16<kN>(raw, hi, lo, code);
                    #pragma unroll
                    for (int i = 0; i < kN; ++i) {
                        const int row = row0 + 2 * S::kTeam * i, col = kTokens + row;
                        const int to = (((chunk / 2) ^ (row & 7)) << 4) + chunk % 2 * 8;
                        *reinterpret_cast<uint2*>(tile + row * 128 + to) = hi[i];
                        *reinterpret_cast<uint2*>(tile + col * 128 + to) = lo[i];
                        if (chunk % 4 == 0) {
                            sf[row * 16 + chunk / 4] = static_cast<uint8_t>(code[i]);
                            sf[col * 16 + chunk / 4] = static_cast<uint8_t>(code[i] == 255 ? 255 : code[i] - 4);
                        }
                    }
                };
                if (S::kPieces == 1 || rows <= 2 * S::kTeam) split(std::integral_constant<int, 1>{});
                else if (S::kPieces == 2 || rows <= 4 * S::kTeam) split(std::integral_constant<int, (S::kPieces < 2 ? 1 : 2)>{});
                else split(std::integral_constant<int, S::kPieces>{});
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(at_stage));
                __syncwarp();
            }
            stage = b_stage;
            phase = b_phase;
            steps += blocks;
        } else if (warp >= 4) {
            // Epilogue: this thread's column of D, the pass's rows of it
            const int rows = at.rows_here(), r0 = at.row;
            const uint32_t quarter = warp % 4, row = quarter * 32 + lane;
            const int n = at.n0 + static_cast<int>(row);
            auto write = [&](int t, float y) {
                if (t >= rows || n >= p.n) return;
                const int64_t to = static_cast<int64_t>(r0 + t) * p.ldd + n;
                y *= p.alpha;
                if (p.d_fp32) {
                    float* const out = static_cast<float*>(p.d) + to;
                    *out = p.accumulate ? *out + y : y;
                } else {
                    __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(p.d) + to;
                    if (p.accumulate) y += __bfloat162float(*out);
                    *out = __float2bfloat16_rn(y);
                }
            };
            if (ok && some) ok = warp_wait(done_bar(accum), accum_phase, ctx, 4);
            tc_fence_after_sync();
            const uint32_t own_rows = S::recv_rows(slices), recv = base + S::kOffRecv;
            float y[kTokens];
            #pragma unroll
            for (int t0 = 0; t0 < kTokens; t0 += 16) {
                // columns hi, lo of 16 rows (of 8: both in one load), the second issuer's added to the first's
                uint32_t v[16], w[16];
                #pragma unroll
                for (int issuer = 0; issuer < S::kIssuers; ++issuer) {
                    const bool mine = kb1 - kb0 > issuer;
                    if (mine) {
                        const uint32_t from = ((quarter * 32) << 16) + accumulators(accum, issuer) + t0;
                        tmem_ld_32x32b_x16(from, v);
                        if constexpr (kTokens >= 16) tmem_ld_32x32b_x16(from + kTokens, w);
                        tmem_ld_wait();
                    }
                    #pragma unroll
                    for (int i = 0; i < (kTokens < 16 ? kTokens : 16); ++i) {
                        const float sum = !mine ? 0.0f : __uint_as_float(v[i]) + __uint_as_float(kTokens >= 16 ? w[i] : v[i + 8]);
                        y[t0 + i] = issuer == 0 ? sum : y[t0 + i] + sum;
                    }
                }
            }
            if (some) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(free_bar(accum));
            }
            __syncwarp();
            if (slices == 1) {
                #pragma unroll
                for (int t = 0; t < kTokens; ++t) write(t, y[t]);
            } else {
                cluster_wait();                                              // every CTA of the cluster may be written to
                uint32_t owner = 0, at_owner = 0;                            // row t of D: CTA t mod slices, its (t / slices)-th
                #pragma unroll
                for (int t = 0; t < kTokens; ++t) {
                    if (t < rows) {
                        st_shared_cluster_u32(map_to_cta(recv + ((rank * own_rows + at_owner) * 128 + row) * 4, owner), __float_as_uint(y[t]));
                        if (++owner == slices) {
                            owner = 0;
                            ++at_owner;
                        }
                    }
                }
                __syncwarp();
                cluster_arrive();                                            // release: what this CTA sent is visible to its owners
                cluster_wait();
                for (uint32_t i = 0; i < own_rows; ++i) {
                    const int t = static_cast<int>(i * slices + rank);
                    if (t >= rows) break;
                    float part[kMaxCluster], sum = 0.0f;                     // (all loads on their way before the first sum)
                    #pragma unroll
                    for (uint32_t s = 0; s < kMaxCluster; ++s)
                        part[s] = s < slices ? __uint_as_float(ld_shared_u32(recv + ((s * own_rows + i) * 128 + row) * 4)) : 0.0f;
                    #pragma unroll
                    for (uint32_t s = 0; s < kMaxCluster; ++s) sum += part[s];
                    write(t, sum);
                }
            }
        }
        __syncwarp();                            // (what follows wants every warp together: lanes beyond N skipped stores)
        if (slices > 1 && (warp < 4 || warp >= 8)) {
            // the other warps only take part in the two barriers of the epilogue
            cluster_wait();
            cluster_arrive();
            cluster_wait();
        }
    }

    __syncthreads();
    if (*abort_flag != 0) {                      // a wait ran out: copies still in flight get time to land
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000) { }
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem, S::kTmemCols);
    }
}

}  // namespace few
}  // namespace dg
