// Attention of prompt chunks over the 8-bit cache on the 5th-generation tensor cores; included by tq_attend8.cu.
//
// A CTA takes 256 query rows (two tiles of 128; rows are token-major, the heads of a group side by side) of one sequence and KV head
// and walks over the keys, 128 tokens at a time:
//
//   planner warp          looks up the blocks and scales of the tiles to come and has their codes copied into shared memory (bulk copies,
//                         2 KB of a page each)
//   converter warps       two for keys, two for values: codes to fp16 - exact, whatever the scale - as operands in shared memory, K K-major,
//                         V MN-major.  (A product in e4m3 itself would need queries and weights as sums of two or three e4m3 terms,
//                         which costs more)
//   product warp          one thread: S_q = Q_q K^T (shared x shared), O_q += P_q V (tensor memory x shared), q = 0, 1
//   softmax warps         two threads for each query row, 64 columns each: weights in fp16 back into columns of S, sums.  (With one
//                         thread a row, two warps a scheduler, their latencies were not covered: 2800 cycles a tile)
//
// The two tiles take turns: while one's weights are computed, the tensor cores work on the other's products.  The references of the softmax
// are raised only when a score passes them by 2^8, so that O in tensor memory is rarely rescaled.  Bound: the exponentials (16 a cycle
// and SM, 2048 cycles a tile pair) next to the products (2048 cycles); conversion and bookkeeping share the issue slots with them.
// Four roles run different code at the same time, and what they repeat has to fit the instruction cache: with everything unrolled (28 KB of
// instructions a step) it missed in 28 % of the cases, the next level was at 77 % of its rate, and a step took 7000 cycles.
// So loops stay loops here, the codes go through shared memory instead of registers, and steps without hidden columns have a
// loop without masks (482 us with one for both).
//
// 32 / 8 heads of 128, bf16: 4 chunks of 700 to 1024 tokens over 1000 to 7168 453 us (658 TFLOP/s; fp16 492), one of 2048 over 16384 730-740
// (790-800), one of 4096 over nothing 213 (646).  A step of two tiles takes 2.6 to 2.9 us, 1.1 of them products: what is left is the chain
// from scores to weights to products and back (one group of eight products by itself 960 to 1120 cycles, 512 of them at work).
// One tile a CTA with two buffers for scores: 580 us, as the codes are then converted for half as many rows.
//
// K's scales enter with the weights, for each 16 columns of the scores: weight = 2^(s c_page + shift_page).  V's enter with the values where they are converted, as far as
// fp16 holds those exactly: 22 powers of two below the largest scale seen so far.  What goes beyond enters with the weights, which
// then use their range whatever the scales are (page_weights in tq_attend8.cu has the same two references m and u); pages 2^(22 + x) below
// the largest lose weights below 2^(x - 32) of the largest, in the product, not in the denominator.
// A NaN in V counts as zero in the product; its dim and token are noted, and rows that see the token become NaN in that dim at the end.
//
// All waits are bounded; one that gives up sets TQ_STATUS_TIMEOUT, every role leaves its loop, copies and products that are under way are waited
// for, and the tensor memory is freed.
#pragma once

#include <type_traits>

namespace tq {
namespace {

// Warps: 0-3 and 4-7 the weights of query tile 0 (columns 0-63, 64-127), 8-11 and 12-15 of tile 1, 16, 17 keys, 18, 19 values, 20 products, 21 planner.
constexpr int kSoftmaxWarps = 16;
constexpr int kPromptThreads = (kSoftmaxWarps + 6) * 32;
constexpr int kTile = 128;                      // query rows of a tile, and tokens of a step
constexpr int kTilePages = kTile / kPageTokens;
constexpr int kPlans = 8;
constexpr int kRankedSeqs = 128;                // sequences that a CTA sorts by length

// The scales of a tile's pages: of K as it is; of V a power of two in two parts, 2^v_exp for the weights and v_factor, fp16 bits, for the values.
struct alignas(16) StepPlan {
    float k_scale[kTilePages], v_exp[kTilePages];
    uint16_t v_factor[kTilePages];
};
// Codes are at most 2^8.8 and multiples of 2^-9: times 2^7 to 2^-15 fp16 holds them exactly.
constexpr int kMostLift = 7, kLeastLift = -15;

template <int D>
struct PromptSmem {
    static constexpr int kOperand = kTile * D * 2;                       // bytes of a tile of queries, keys or values
    static constexpr int kBars = 0;
    static constexpr int kTmemSlot = 288;
    static constexpr int kFlags = 292;                                   // failed, NaN seen
    static constexpr int kPlan = 304;
    static constexpr int kNan = kPlan + kPlans * sizeof(StepPlan);       // [D] first token with a NaN in this dim of V
    static constexpr int kOver = kNan + D * 4;                           // [2 steps][8 pairs of warps][2] a score passes its reference
    static constexpr int kRows = kOver + 2 * 8 * 2 * 4;                  // [8 pairs][32] one value of a row, from thread to thread
    static constexpr int kQ = 2688;                                      // [2]
    static constexpr int kK = kQ + 2 * kOperand;                         // [2]
    static constexpr int kV = kK + 2 * kOperand;                         // [2]
    static constexpr int kRawK = kV + 2 * kOperand;                      // codes of a tile's keys, values
    static constexpr int kRawV = kRawK + kTile * D;
    static constexpr int kBytes = kRawV + kTile * D;
    static_assert(kPlan % 16 == 0 && kRows + 8 * 32 * 4 <= kQ && kBytes <= 227 * 1024, "shared memory map");
};

enum PromptBar { kbKFull = 0, kbKEmpty = 2, kbVFull = 4, kbVEmpty = 6, kbSFull = 8, kbPFull = 10, kbPvDone = 12, kbRawKFull = 14, kbRawKEmpty = 15, kbRawVFull = 16, kbRawVEmpty = 17,
                 kbPlanFull = 18, kbPlanEmpty = 18 + kPlans, kbDrained = 18 + 2 * kPlans, kbBars };
static_assert(kbBars * 8 <= 288, "barriers");

__device__ __forceinline__ void prompt_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void prompt_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void prompt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void prompt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void prompt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void prompt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor without swizzle: 8 x 16-byte core matrices; lbo, sbo in bytes.
__device__ __forceinline__ uint64_t prompt_desc(uint32_t at, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((at & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) | (static_cast<uint64_t>(sbo >> 4) << 32) | (1ull << 46);
}
// kind::f16, fp16 x fp16 -> fp32, M = 128
__host__ __device__ constexpr uint32_t prompt_idesc(int n, int b_mn_major) {
    return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void prompt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void prompt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void prompt_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at) : "memory");
}
__device__ __forceinline__ void prompt_st32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void prompt_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// two fp32 in one register pair
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What all roles of a CTA agree on.
struct PromptJob {
    int first_row, kvh, r0, nrows, tiles;       // tiles: of query rows, 1 or 2
    int len, nq;
    int token_a, token_b;                       // tokens that this CTA walks over
};

// 16 codes as fp16 into two 16-byte pieces.
template <bool SCALED>
__device__ __forceinline__ void convert16(uint4 codes, uint32_t at, uint32_t step, uint32_t factor) {
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = e4m3x2_to_half2(w[i] & 0xffffu);
        h[2 * i + 1] = e4m3x2_to_half2(w[i] >> 16);
        if (SCALED) {
            asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[2 * i]) : "r"(factor));
            asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[2 * i + 1]) : "r"(factor));
        }
    }
    sts16(at, h[0], h[1], h[2], h[3]);
    sts16(at + step, h[4], h[5], h[6], h[7]);
}

// A whole warp's wait, with one answer for the warp: what follows it is for whole warps.  A role leaves at its own first wait that gives up;
// those that wait for it give up after it.
__device__ __forceinline__ bool waited(uint64_t* bar, uint32_t parity, volatile int* flags) {
    const bool ok = mbar_wait_bounded(bar, parity);
    if (!ok) flags[0] = 1;
    return __all_sync(0xffffffffu, ok);
}

// Lane i < 8 looks at page i of a tile, and has its keys copied, lane 8 + i its values.
template <int D>
__device__ void prompt_plan(const Attend8Params& p, const PromptJob& job, int seq, uint8_t* smem, uint64_t* bars, volatile int* flags) {
    using Smem = PromptSmem<D>;
    constexpr uint32_t kPart = kPageTokens * D;
    const int lane = threadIdx.x & 31, mine = lane & 7;
    const int32_t* table = p.tables + seq * p.table_stride;
    const int pages = pages_of_length(job.token_b);
    StepPlan* plans = reinterpret_cast<StepPlan*>(smem + Smem::kPlan);
    bool bad = false;
    auto ask_block = [&](int token0) {
        const int page = token0 / kPageTokens + mine;
        return page < pages ? __ldg(table + page / p.pages_per_block) : 0;
    };
    int block = ask_block(job.token_a), step = 0, keys = 0, values = 0;     // copies of tiles that were issued
    int largest = kMinExponent - kMostLift;                                 // scale of V so far
    for (int token0 = job.token_a; token0 < job.token_b; token0 += kTile, ++step) {
        const int page = token0 / kPageTokens + mine, count = min(pages - token0 / kPageTokens, kTilePages);
        const bool here = mine < count;
        if (here && (block < 0 || block >= p.num_blocks)) {
            bad = true;
            block = block < 0 ? 0 : static_cast<int>(p.num_blocks - 1);
        }
        const uint8_t* at = here ? page_address<D>(p, page, block, job.kvh) : nullptr;
        block = ask_block(token0 + kTile);
        const float2 scales = here ? __ldg(reinterpret_cast<const float2*>(at + cache8_scale_off(D))) : make_float2(0.f, 0.f);
        const int ev = static_cast<int>(__float_as_uint(scales.y) >> 23 & 0xffu) - 127;
        largest = max(largest, __reduce_max_sync(0xffffffffu, here ? ev : kMinExponent - kMostLift));
        const int lift = here ? max(ev - largest + kMostLift, kLeastLift) : 0;
        // Pages that are not there keep the codes of another tile: their columns are masked, and finite values times zero are zero.
        const uint32_t turn = (step & 1) ^ 1;
        if (!waited(bars + kbRawKEmpty, turn, flags)) break;
        if (lane == 0) mbar_expect_tx(bars + kbRawKFull, count * kPart);
        __syncwarp();
        if (here && lane < 8) bulk_g2s(smem + Smem::kRawK + mine * kPart, at, kPart, bars + kbRawKFull);
        ++keys;
        const int slot = step % kPlans;
        if (!waited(bars + kbPlanEmpty + slot, (step / kPlans & 1) ^ 1, flags) || !waited(bars + kbRawVEmpty, turn, flags)) break;
        StepPlan& plan = plans[slot];
        if (lane < kTilePages) {
            plan.k_scale[mine] = scales.x;
            plan.v_exp[mine] = static_cast<float>(here ? ev - lift : largest - kMostLift);
            plan.v_factor[mine] = static_cast<uint16_t>(lift == kLeastLift ? 0x200 : (lift + 15) << 10);
        }
        __syncwarp();
        if (lane == 0) {
            prompt_arrive(bars + kbPlanFull + slot);
            mbar_expect_tx(bars + kbRawVFull, count * kPart);
        }
        __syncwarp();
        if (here && lane >= 8 && lane < 16) bulk_g2s(smem + Smem::kRawV + mine * kPart, at + kPart, kPart, bars + kbRawVFull);
        ++values;
    }
    // Nothing is on its way to shared memory when the CTA leaves it, also where the converters have given up.
    if (keys && !mbar_wait_bounded(bars + kbRawKFull, (keys - 1) & 1)) flags[0] = 1;
    if (values && !mbar_wait_bounded(bars + kbRawVFull, (values - 1) & 1)) flags[0] = 1;
    if (bad && p.status) atomicOr(p.status, TQ_STATUS_BAD_BLOCK);
}

// A warp converts 4 pages of a tile, keys or values.
template <int D, bool VALUES>
__device__ void prompt_convert(const PromptJob& job, uint8_t* smem, uint64_t* bars, volatile int* flags) {
    using Smem = PromptSmem<D>;
    constexpr int kLoads = D / 32, kPages = kTilePages / 2;                 // 16-byte pieces of a lane and page
    // K: 16 bytes (8 dims) of 128 tokens side by side.  V: of 8 tokens, then the next 8 dims, then the next 8 tokens.
    constexpr uint32_t kColumn = VALUES ? 128 : 2048;
    constexpr int kFull = VALUES ? kbVFull : kbKFull, kEmpty = VALUES ? kbVEmpty : kbKEmpty;
    constexpr int kRawFull = VALUES ? kbRawVFull : kbRawKFull, kRawEmpty = VALUES ? kbRawVEmpty : kbRawKEmpty;
    const int lane = threadIdx.x & 31, first = (threadIdx.x >> 5 & 1) * kPages;
    // A lane turns pieces (token, 2 j + half); the tokens of 8 lanes start on different banks where it stores, and where it loads the
    // pieces of odd tokens are taken in another order
    const int tok = lane & 15, half = lane >> 4;
    const uint32_t base = smem_u32(smem), operand = base + (VALUES ? Smem::kV : Smem::kK), raw = base + (VALUES ? Smem::kRawV : Smem::kRawK);
    int* first_nan = reinterpret_cast<int*>(smem + Smem::kNan);
    const StepPlan* plans = reinterpret_cast<const StepPlan*>(smem + Smem::kPlan);      // written before the copy of the values is asked for
    int step = 0;
    for (int token0 = job.token_a; token0 < job.token_b; token0 += kTile, ++step) {
        const int s = step & 1;
        if (!waited(bars + kRawFull, step & 1, flags) || !waited(bars + kEmpty + s, (step >> 1 & 1) ^ 1, flags)) return;
#pragma unroll 1
        for (int i = 0; i < kPages; ++i) {
            const int token = (first + i) * kPageTokens + tok;
            const uint32_t to = operand + s * Smem::kOperand + (VALUES ? (token >> 3) * (D * 16) + (token & 7) * 16 : token * 16);
            const uint32_t factor = VALUES ? plans[step % kPlans].v_factor[first + i] * 0x10001u : 0u;
            uint4 x[kLoads];
            uint32_t nan = 0;                                               // bit 7 of a byte: a code is 0x7f or 0xff
#pragma unroll
            for (int j = 0; j < kLoads; ++j) x[j] = lds16(raw + token * D + ((2 * j + half) ^ (tok & (2 * kLoads - 1))) * 16);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                if (VALUES)
                    nan |= ((x[j].x & 0x7f7f7f7fu) + 0x01010101u) | ((x[j].y & 0x7f7f7f7fu) + 0x01010101u) |
                           ((x[j].z & 0x7f7f7f7fu) + 0x01010101u) | ((x[j].w & 0x7f7f7f7fu) + 0x01010101u);
                convert16<VALUES>(x[j], to + ((2 * j + half) ^ (tok & (2 * kLoads - 1))) * 2 * kColumn, kColumn, factor);
            }
            if (VALUES && (nan & 0x80808080u)) {
                // rare: this lane's pieces once more, from where they were put
                flags[1] = 1;
                asm volatile("" ::: "memory");
#pragma unroll 1
                for (int j = 0; j < kLoads * 16; ++j) {
                    const int dim = ((2 * (j >> 4) + half) ^ (tok & (2 * kLoads - 1))) * 16 + (j & 15);
                    uint16_t* at = reinterpret_cast<uint16_t*>(smem + (to - base) + (dim >> 3) * 128 + (dim & 7) * 2);
                    if ((*at & 0x7fffu) > 0x7c00u) {
                        *at = 0;
                        atomicMin(first_nan + dim, token0 + token);
                    }
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            prompt_arrive(bars + kRawEmpty);
            prompt_arrive(bars + kFull + s);
        }
    }
}

__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// The whole warp walks through the steps, so that addresses and descriptors stay in uniform registers, and one lane issues.  (With a
// single lane walking, the eight products of an operand took 1200 cycles to issue; they take 512 to run.)  All 512 columns
// are this CTA's, so that they begin at address 0.
template <int D>
__device__ void prompt_multiply(const PromptJob& job, uint8_t* smem, uint64_t* bars, volatile int* flags) {
    using Smem = PromptSmem<D>;
    constexpr uint32_t kScores = prompt_idesc(kTile, 0), kOut = prompt_idesc(D, 1);
    const uint32_t base = smem_u32(smem);
    const int steps = __shfl_sync(0xffffffffu, (job.token_b - job.token_a + kTile - 1) / kTile, 0);
    const bool both = __shfl_sync(0xffffffffu, job.tiles, 0) == 2;
    auto wait = [&](int bar, uint32_t parity) { return waited(bars + bar, parity, flags); };
    const uint64_t queries = prompt_desc(base + Smem::kQ, 2048, 128), keys = prompt_desc(base + Smem::kK, 2048, 128),
                   values = prompt_desc(base + Smem::kV, D * 16, 128);
    auto scores = [&](int q, int s) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            prompt_mma_ss(q * kTile, queries + (q * Smem::kOperand + i * 4096) / 16, keys + (s * Smem::kOperand + i * 4096) / 16, kScores, i ? 1u : 0u);
        prompt_commit(bars + kbSFull + q);
    };
    auto products = [&](int q, int s, uint32_t accumulate) {
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i)
            prompt_mma_ts(2 * kTile + q * kTile, q * kTile + i / 4 * 64 + i % 4 * 8, values + (s * Smem::kOperand + i * 2 * (D * 16)) / 16, kOut, i ? 1u : accumulate);
        prompt_commit(bars + kbPvDone + q);
    };
    auto walk = [&]() {
        if (!wait(kbKFull, 0)) return;
        prompt_fence_after();
        if (elect_one()) {
            scores(0, 0);
            if (both) scores(1, 0);
            prompt_commit(bars + kbKEmpty);
        }
        __syncwarp();
        for (int step = 0; step < steps; ++step) {
            const int s = step & 1, n = s ^ 1;
            const bool more = step + 1 < steps;
            if (!wait(kbVFull + s, step >> 1 & 1)) return;
            if (!wait(kbPFull, step & 1)) return;
            prompt_fence_after();
            if (elect_one()) {
                products(0, s, step ? 1u : 0u);
                if (!both) {
                    prompt_commit(bars + kbVEmpty + s);
                    prompt_commit(bars + kbPlanEmpty + step % kPlans);
                }
            }
            __syncwarp();
            if (more) {
                if (!wait(kbKFull + n, (step + 1) >> 1 & 1)) return;
                prompt_fence_after();
                if (elect_one()) {
                    scores(0, n);
                    if (!both) prompt_commit(bars + kbKEmpty + n);
                }
                __syncwarp();
            }
            if (!both) continue;
            if (!wait(kbPFull + 1, step & 1)) return;
            prompt_fence_after();
            if (elect_one()) {
                products(1, s, step ? 1u : 0u);
                prompt_commit(bars + kbVEmpty + s);
                prompt_commit(bars + kbPlanEmpty + step % kPlans);              // the softmax warps are done with it, too
                if (more) {
                    scores(1, n);
                    prompt_commit(bars + kbKEmpty + n);
                }
            }
            __syncwarp();
        }
    };
    walk();
    // No product is under way when tensor memory is freed, also where the softmax warps have given up.
    if (elect_one()) prompt_commit(bars + kbDrained);
    __syncwarp();
    wait(kbDrained, 0);
}

constexpr float kFarApart = 60.f;           // values so many powers of two below the reference: fp32 may not hold the weights in its units

// What a weight counts for in the denominator where the values lie further below the reference than the product's fp16 goes: as it was rounded, or, where
// fp16 has no full precision (2^-14), as it is.
__device__ __forceinline__ float counted(float weight, float rounded) { return weight < 6.103515625e-5f ? weight : rounded; }

constexpr float kTiny = 1e-38f;             // factors of scores are never zero: times -inf that would be NaN

// Columns from `visible` on see nothing.
__device__ __forceinline__ void hide(uint32_t* x, int visible) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i >= visible) x[i] = 0xff800000u;
}

// A value of the other thread of this row.  The pair's warps meet at a barrier of their own before and after.
__device__ __forceinline__ float exchange(float* row, int half, int barrier, float mine) {
    float theirs = 0.f;
    if (half) *row = mine;
    asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory");
    if (!half) {
        theirs = *row;
        *row = mine;
    }
    asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory");
    if (half) theirs = *row;
    asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory");
    return theirs;
}

template <int D, bool BF16>
__device__ void prompt_softmax(const Attend8Params& p, const PromptJob& job, int split, uint8_t* smem, uint64_t* bars, volatile int* flags, uint32_t tmem,
                               float row_scale) {
    using Smem = PromptSmem<D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = warp >> 3, half = warp >> 2 & 1, together = q * 4 + (warp & 3);
    const int row = job.r0 + q * kTile + (warp & 3) * 32 + lane;
    const int limit = job.len - job.nq + min(row, job.nrows - 1) / p.group + 1;
    const int warp_limit = __reduce_min_sync(0xffffffffu, limit);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + q * kTile + 64 * half, o_at = tmem + lanes + 2 * kTile + q * kTile + D / 2 * half;
    const StepPlan* plans = reinterpret_cast<const StepPlan*>(smem + Smem::kPlan);
    volatile int* over = reinterpret_cast<volatile int*>(smem + Smem::kOver) + together * 2;
    float* row_slot = reinterpret_cast<float*>(smem + Smem::kRows) + together * 32 + lane;
    float m = kNothing, u = kNothing, l = 0.f;
    bool ok = true;
    int step = 0;
    for (int token0 = job.token_a; token0 < job.token_b; token0 += kTile, ++step) {
        bool lost = !waited(bars + kbPlanFull + step % kPlans, step / kPlans & 1, flags);
        lost |= !waited(bars + kbSFull + q, step & 1, flags);
        prompt_fence_after();
        const StepPlan& plan = plans[step % kPlans];
        const int visible = limit - token0 - 64 * half;
        const bool masked = token0 + kTile > warp_limit;
        // Weights are computed against the references as they are, and the largest scores on the way.  Only where these pass the
        // references - always at first - the references are raised, and the scores, which are still there, gone through again.
        float sum;
        bool far;
        uint32_t w[32];
        for (bool again = false;; again = true) {
            float most = kNothing, most_v = kNothing;
            // Twice, so that the code for columns that see nothing does not lie in the way of the steps that have none.
            auto pass = [&](auto cut) {
                sum = 0.f;
                far = false;
                uint32_t x[2][16];
                prompt_ld16(s_at, x[0]);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t(&of)[16] = x[g & 1];
                    prompt_wait_ld();
                    if (g < 3) prompt_ld16(s_at + 16 * g + 16, x[(g + 1) & 1]);
                    if constexpr (decltype(cut)::value) hide(of, visible - 16 * g);
                    const float c = fmaxf(row_scale * plan.k_scale[4 * half + g], kTiny), ev = plan.v_exp[4 * half + g], shift = ev + kHeadroom - u;
                    float a = fmaxf(fmaxf(__uint_as_float(of[0]), __uint_as_float(of[1])), __uint_as_float(of[2]));
#pragma unroll
                    for (int i = 3; i < 15; i += 2) a = fmaxf(fmaxf(a, __uint_as_float(of[i])), __uint_as_float(of[i + 1]));
                    a = fmaxf(a, __uint_as_float(of[15])) * c;
                    most = fmaxf(most, a);
                    most_v = fmaxf(most_v, a + ev);
                    const uint64_t c2 = pair(c, c), shift2 = pair(shift, shift);
                    uint64_t sums = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float y, z;
                        unpair(fma2(pair(__uint_as_float(of[2 * i]), __uint_as_float(of[2 * i + 1])), c2, shift2), y, z);
                        y = ex2(y);
                        z = ex2(z);
                        w[8 * g + i] = pack_half2(y, z);
                        if (!BF16) {
                            // as they are rounded for the product (page_weights); an output in bf16 does not show the difference
                            const float2 v = unpack_half2(w[8 * g + i]);
                            y = decltype(cut)::value ? counted(y, v.x) : v.x;
                            z = decltype(cut)::value ? counted(z, v.y) : v.y;
                        }
                        sums = add2(sums, pair(y, z));
                    }
                    float sum0, sum1;
                    unpair(sums, sum0, sum1);
                    const float up = u - ev - m;
                    far |= up > kFarApart;
                    sum = fmaf(sum0 + sum1, up > kFarApart ? 0.f : ex2(up - kHeadroom), sum);   // in units of m again
                }
            };
            // the rarer code also looks at what each weight counts for
            bool apart = false;
            if constexpr (!BF16) {
                const float4 ev = *reinterpret_cast<const float4*>(plan.v_exp + 4 * half);
                apart = __any_sync(0xffffffffu, u - m - fminf(fminf(ev.x, ev.y), fminf(ev.z, ev.w)) > kLossless);
            }
            if (masked || apart) pass(std::true_type{});
            else pass(std::false_type{});
            if (again) break;
            // Both warps of the rows decide alike, also about giving up.
            const int mine = __any_sync(0xffffffffu, most > m + kLazy || most_v > u + kLazy) ? 1 : 0;
            if (lane == 0) over[(step & 1) * 16 + half] = mine | (lost ? 2 : 0);
            __syncwarp();
            asm volatile("bar.sync %0, 64;" ::"r"(1 + together) : "memory");
            const int both = over[(step & 1) * 16] | over[(step & 1) * 16 + 1];
            if (both & 2) ok = false;
            if (both != 1) break;
            most = fmaxf(most, exchange(row_slot, half, 1 + together, most));
            most_v = fmaxf(most_v, exchange(row_slot, half, 1 + together, most_v));
            const float m1 = fmaxf(m, most), u1 = fmaxf(u, most_v);
            l *= ex2(m - m1);
            const float down = ex2(u - u1);
            m = m1;
            u = u1;
            if (step) {
                // O is whole when the product of the step before is done
                waited(bars + kbPvDone + q, (step - 1) & 1, flags);
                prompt_fence_after();
#pragma unroll 1
                for (int h = 0; h < D / 32; ++h) {
                    uint32_t o[16];
                    prompt_ld16(o_at + 16 * h, o);
                    prompt_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
                    prompt_st16(o_at + 16 * h, o);
                }
            }
        }
        if (!ok) break;
        if (__any_sync(0xffffffffu, far)) {
            // Value scales so far apart that fp32 may not hold the weights in units of u: those columns are read again.
#pragma unroll 1
            for (int g = 0; g < 4; ++g) {
                uint32_t of[16];
                prompt_ld16(s_at + 16 * g, of);
                prompt_wait_ld();
                hide(of, visible - 16 * g);
                const float c = fmaxf(row_scale * plan.k_scale[4 * half + g], kTiny);
                float more = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) more += ex2(fmaf(__uint_as_float(of[i]), c, -m));
                if (u - plan.v_exp[4 * half + g] - m > kFarApart) sum += more;
            }
        }
        l += sum;
        prompt_st32(s_at, w);
        prompt_wait_st();
        prompt_fence_before();
        __syncwarp();
        if (lane == 0) prompt_arrive(bars + kbPFull + q);
    }
    if (ok && step) {
        ok = waited(bars + kbPvDone + q, (step - 1) & 1, flags);
        prompt_fence_after();
    }
    __syncwarp();
    ok = ok && __all_sync(0xffffffffu, flags[0] == 0);
    asm volatile("bar.sync %0, 64;" ::"r"(1 + together) : "memory");
    l += exchange(row_slot, half, 1 + together, l);
    // The row's values: in units of the weights' reference, divided by their sum where this CTA saw all of them.
    const bool whole = p.chunks == 1, store = ok && row < job.nrows;
    const int token = row / p.group, head = job.kvh * p.group + row - token * p.group;
    const int64_t at = static_cast<int64_t>(job.first_row + token) * p.q_heads + head;
    float f = l == 0.f ? 0.f : ex2(u - m - kHeadroom);
    if (whole && l != 0.f) f /= l;
    const bool nothing = job.token_a >= job.token_b || l == 0.f;
    const int* first_nan = reinterpret_cast<const int*>(smem + Smem::kNan);
#pragma unroll 1
    for (int h = 0; h < D / 32; ++h) {
        const int d0 = D / 2 * half + 16 * h;
        uint32_t x[16];
        if (job.token_a < job.token_b && ok) {
            prompt_ld16(o_at + 16 * h, x);
            prompt_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = nothing ? 0u : __float_as_uint(__uint_as_float(x[i]) * f);
        if (flags[1]) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (first_nan[d0 + i] < limit) x[i] = 0x7fffffffu;
        }
        if (!store) continue;
        if (whole) {
            uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at * D + d0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = pack_out(__uint_as_float(x[8 * i + 2 * j]), __uint_as_float(x[8 * i + 2 * j + 1]), BF16);
                to[i] = make_uint4(v[0], v[1], v[2], v[3]);
            }
        } else {
            float2* to = reinterpret_cast<float2*>(p.partials + (at * p.chunks + split) * (D + 2) + d0);
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i] = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
        }
    }
    if (store && !whole && !half) *reinterpret_cast<float2*>(p.partials + (at * p.chunks + split) * (D + 2) + D) = make_float2(m, l);
}

// Queries of a tile as K-major A operand, two threads a row; returns the factor of its scores in units of log2.  All threads of the block
// come here (a row's largest value is looked for by both of its threads), those of no row with row = -1.
template <int D, bool BF16>
__device__ float prompt_queries(const Attend8Params& p, const PromptJob& job, uint8_t* smem) {
    using Smem = PromptSmem<D>;
    constexpr int kWords = D / 4;
    const int warp = threadIdx.x >> 5, q = warp >> 3, half = warp >> 2 & 1, r = threadIdx.x & (kTile - 1), row = job.r0 + q * kTile + r;
    const bool mine = warp < 8 * job.tiles;
    uint32_t* largest = reinterpret_cast<uint32_t*>(smem + Smem::kK);       // not in use yet
    uint32_t x[kWords];
    uint32_t most = 0;
    if (mine && row < job.nrows) {
        const int token = row / p.group, head = job.kvh * p.group + row - token * p.group;
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(job.first_row + token) * p.q_heads + head) * D +
                                                           D / 2 * half);
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const uint4 w = __ldg(from + i);
            x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = 0;
    }
    if constexpr (BF16) {      // into the range of fp16 by a power of two, as in load_queries
#pragma unroll
        for (int i = 0; i < kWords; ++i) most = max(most, max(x[i] & 0x7fffu, x[i] >> 16 & 0x7fffu));
        if (mine) largest[threadIdx.x] = most;
        __syncthreads();
        if (mine) most = max(most, largest[threadIdx.x ^ kTile]);
        __syncthreads();
    }
    if (!mine) return 0.f;
    float row_scale = fabsf(p.scale_log2);
    if constexpr (BF16) {
        const int e = min(max(static_cast<int>(most >> 7) - 127, -120), 120);
        const float down = exp2_int(-e);
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = pack_half2(__uint_as_float(x[i] << 16) * down, __uint_as_float(x[i] & 0xffff0000u) * down);
        row_scale *= exp2_int(e);
    }
    const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    const uint32_t to = smem_u32(smem) + Smem::kQ + q * Smem::kOperand + r * 16 + half * (D / 16) * 2048;
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) sts16(to + i * 2048, x[4 * i] ^ sign, x[4 * i + 1] ^ sign, x[4 * i + 2] ^ sign, x[4 * i + 3] ^ sign);
    return row_scale;
}

// The sequence and its block of 256 query rows that slot `slot` stands for, -1 when there are fewer.  Only blocks that exist get a slot, so
// that a batch of decodes with one chunk does not launch a CTA for every block that a decode could have had.  CTAs start in the
// order of the slots: a sequence's blocks from the last one, which sees the most, down, and the longest sequence first, so that
// the last CTAs are short: 16 uneven sequences 316 us (362 unsorted), 4 chunks of 700 to 1024 tokens 441 (453).
__device__ __forceinline__ void prompt_place(const Attend8Params& p, int slot, int* shared, int& seq, int& block) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto blocks_of = [&](int s) {
        int first_row, nq;
        rows_of(p, s, first_row, nq);
        return nq * p.group <= p.small_rows ? 0 : (nq * p.group + 2 * kTile - 1) / (2 * kTile);
    };
    auto take = [&](int s, uint32_t place, int blocks) {
        if (place >= static_cast<uint32_t>(blocks)) return;
        shared[0] = s;
        shared[1] = blocks - 1 - static_cast<int>(place);
    };
    if (tid == 0) shared[0] = -1;
    if (p.seqs <= kRankedSeqs) {
        int2* all = reinterpret_cast<int2*>(shared + 2);                    // lengths, blocks
        const int2 mine = tid < p.seqs ? make_int2(p.seq_lens[tid], blocks_of(tid)) : make_int2(0, 0);
        if (tid < p.seqs) all[tid] = mine;
        __syncthreads();
        if (mine.y) {
            uint32_t before = 0;
            for (int i = 0; i < p.seqs; ++i) before += all[i].x > mine.x || (all[i].x == mine.x && i < tid) ? all[i].y : 0;
            take(tid, slot - before, mine.y);
        }
    } else {
        const int each = (p.seqs + kPromptThreads - 1) / kPromptThreads, first = tid * each;
        uint32_t sum = 0;
        for (int s = first; s < min(first + each, p.seqs); ++s) sum += blocks_of(s);
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += y;
        }
        if (lane == 31) shared[2 + warp] = before;
        __syncthreads();
        before -= sum;
        for (int w = 0; w < warp; ++w) before += shared[2 + w];
        for (int s = first; s < min(first + each, p.seqs); ++s) {
            const int blocks = blocks_of(s);
            take(s, slot - before, blocks);
            before += blocks;
        }
    }
    __syncthreads();
    // By a shuffle, so that the compiler knows them to be the same for a warp (2048 tokens over 16384: 718 to 725 us, 731 without).
    seq = __shfl_sync(0xffffffffu, shared[0], 0);
    block = __shfl_sync(0xffffffffu, shared[1], 0);
    __syncthreads();                                                        // before queries take this place
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPromptThreads, 1) attend8_prompt_kernel(const Attend8Params p) {
    using Smem = PromptSmem<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
    volatile int* flags = reinterpret_cast<volatile int*>(smem + Smem::kFlags);
    const int tid = threadIdx.x, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + kbKFull + i, 2);
            mbar_init(bars + kbKEmpty + i, 1);
            mbar_init(bars + kbVFull + i, 2);
            mbar_init(bars + kbVEmpty + i, 1);
            mbar_init(bars + kbSFull + i, 1);
            mbar_init(bars + kbPFull + i, 8);
            mbar_init(bars + kbPvDone + i, 1);
        }
        mbar_init(bars + kbDrained, 1);
        mbar_init(bars + kbRawKFull, 1);
        mbar_init(bars + kbRawKEmpty, 2);
        mbar_init(bars + kbRawVFull, 1);
        mbar_init(bars + kbRawVEmpty, 2);
        for (int i = 0; i < kPlans; ++i) {
            mbar_init(bars + kbPlanFull + i, 1);
            mbar_init(bars + kbPlanEmpty + i, 1);
        }
        flags[0] = flags[1] = 0;
        fence_barrier_init();
    }
    for (int i = tid; i < D; i += kPromptThreads) reinterpret_cast<int*>(smem + Smem::kNan)[i] = INT32_MAX;
    pdl_wait();
    pdl_release();

    // Splits of one block of rows side by side, then the KV heads, then the blocks of rows.
    int rest = blockIdx.x;
    const int split = rest % p.chunks;
    rest /= p.chunks;
    PromptJob job;
    job.kvh = rest % p.kv_heads;
    int seq, block;
    prompt_place(p, rest / p.kv_heads, reinterpret_cast<int*>(smem + Smem::kQ), seq, block);
    if (p.zero_rest && blockIdx.x == 0) zero_ends<D>(p);
    if (p.status && blockIdx.x == 0) {
        for (int s = tid; s < p.seqs; s += kPromptThreads) {
            const bool left_out = rows_of(p, s, job.first_row, job.nq) > 0, too_long = pages_of_length(p.seq_lens[s]) > p.max_pages;
            if (left_out || too_long) atomicOr(p.status, (too_long ? TQ_STATUS_BAD_BLOCK : 0) | (left_out ? TQ_STATUS_TOO_LONG : 0));
        }
    }
    if (seq < 0) return;
    const int left_out = rows_of(p, seq, job.first_row, job.nq);
    if (left_out && p.zero_rest && block == 0 && split == 0 && job.kvh == 0) zero_rows<D>(p, job.first_row + job.nq, job.first_row + job.nq + left_out);
    job.nrows = job.nq * p.group;
    job.r0 = block * 2 * kTile;
    job.len = p.seq_lens[seq];
    if (pages_of_length(job.len) > p.max_pages) job.len = p.max_pages * kPageTokens;
    job.tiles = job.nrows - job.r0 > kTile ? 2 : 1;
    const int most = max(job.len - job.nq + min(job.r0 + 2 * kTile - 1, job.nrows - 1) / p.group + 1, 0);
    const int steps = (most + kTile - 1) / kTile, each = (steps + p.chunks - 1) / p.chunks;
    job.token_a = min(split * each * kTile, most);
    job.token_b = min((split + 1) * each * kTile, most);

    if (warp == kSoftmaxWarps + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem) + Smem::kTmemSlot), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const float row_scale = prompt_queries<D, BF16>(p, job, smem);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prompt_fence_before();
    __syncthreads();
    prompt_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + Smem::kTmemSlot);
    if (warp < kSoftmaxWarps) {
        if (warp < 8 * job.tiles) prompt_softmax<D, BF16>(p, job, split, smem, bars, flags, tmem, row_scale);
    } else if (warp < kSoftmaxWarps + 2) {
        prompt_convert<D, false>(job, smem, bars, flags);
    } else if (warp < kSoftmaxWarps + 4) {
        prompt_convert<D, true>(job, smem, bars, flags);
    } else if (warp == kSoftmaxWarps + 5) {
        prompt_plan<D>(p, job, seq, smem, bars, flags);
    } else if (job.token_a < job.token_b) {
        prompt_multiply<D>(job, smem, bars, flags);
    }
    __syncwarp();
    if (flags[0] && p.status && (tid & 31) == 0) atomicOr(p.status, TQ_STATUS_TIMEOUT);
    prompt_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace
}  // namespace tq
