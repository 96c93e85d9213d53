// Attention of prompt chunks over the 8-bit cache on the 5th-generation tensor cores; included by tq_attend8.cu.
//
// A CTA takes 256 query rows (two tiles of 128; rows are token-major, the heads of a group side by side) of one sequence and KV head
// and walks over the keys, 128 tokens at a time:
//
//   converter warps 8-11  read the codes of a tile's 8 pages (16 bytes a lane), bring pages to one power-of-two scale while they
//                         turn them into fp16 - exact, e4m3 has 4 significant bits - and write both operands into shared memory:
//                         K as K-major B operand, V as MN-major one.  An earlier form of the product in e4m3 itself would
//                         need the queries and weights as sums of two or three e4m3 terms, which costs more than the conversion
//   MMA warp 12           one thread: S_q = Q_q K^T (shared x shared), O_q += P_q V (tensor memory x shared), q = 0, 1
//   softmax warps 0-3, 4-7  thread = query row of tile 0 / 1: maximum, weights in fp16 back into the columns of S, sums
//
// The two tiles take turns: while one's weights are computed, the tensor cores work on the other's products.  The references of the softmax
// are raised only when a score passes them by 2^8, so that O in tensor memory is rarely rescaled.  Bound: the exponentials (16 a cycle
// and SM, 2048 cycles a tile pair) next to the products (2048 cycles); conversion and bookkeeping share the issue slots with them.
//
// Scales of V that are far apart: fp16 holds codes exactly for pages within 2^15 of the tile's largest scale.  A tile with more is walked
// over several times, each time with the pages of one range (others masked), so that no page's values lose bits to another's.
// A NaN in V counts as zero in the product; its dim and token are noted, and rows that see the token become NaN in that dim at the end.
//
// All waits are bounded; one that gives up sets TQ_STATUS_TIMEOUT, every role leaves its loop and the tensor memory is freed.
#pragma once

namespace tq {
namespace {

constexpr int kPromptThreads = 13 * 32;
constexpr int kTile = 128;                      // query rows of a tile, and tokens of a step
constexpr int kTilePages = kTile / kPageTokens;
constexpr int kDescs = 4;

struct StepDesc {
    int token0, mask, last, v_exp;
    float k_scale;
    int pad[3];
};

template <int D>
struct PromptSmem {
    static constexpr int kOperand = kTile * D * 2;                       // bytes of a tile of queries, keys or values
    static constexpr int kBars = 0;
    static constexpr int kTmemSlot = 128;
    static constexpr int kFlags = 132;                                   // failed, NaN seen
    static constexpr int kDesc = 144;
    static constexpr int kNan = kDesc + kDescs * 32;                     // [D] first token with a NaN in this dim of V
    static constexpr int kQ = 1024;                                      // [2]
    static constexpr int kK = kQ + 2 * kOperand;                         // [2]
    static constexpr int kV = kK + 2 * kOperand;                         // [2]
    static constexpr int kBytes = kV + 2 * kOperand;
    static_assert(kNan + D * 4 <= kQ, "shared memory map");
};

enum PromptBar { kbKFull = 0, kbKEmpty = 2, kbVFull = 4, kbVEmpty = 6, kbSFull = 8, kbPFull = 10, kbPvDone = 12 };

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
__device__ __forceinline__ void prompt_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
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

__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What all roles of a CTA agree on.
struct PromptJob {
    int first_row, kvh, r0, nrows, tiles;       // tiles: of query rows, 1 or 2
    int len, nq;
    int token_a, token_b;                       // tokens that this CTA walks over
};

// 16 codes times 2^d, as fp16, into two 16-byte pieces.
template <bool VALUES>
__device__ __forceinline__ void convert16(uint4 codes, uint32_t factor, bool plain, uint32_t at, uint32_t step) {
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = e4m3x2_to_half2(w[i] & 0xffffu);
        h[2 * i + 1] = e4m3x2_to_half2(w[i] >> 16);
    }
    if (!plain) {
        const __half2 f = *reinterpret_cast<const __half2*>(&factor);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), f);
            h[i] = *reinterpret_cast<const uint32_t*>(&x);
        }
    }
    sts16(at, h[0], h[1], h[2], h[3]);
    sts16(at + step, h[4], h[5], h[6], h[7]);
}

// 2^d as half2: exact down to 2^-24, zero below
__device__ __forceinline__ uint32_t half2_power(int d) {
    const uint32_t h = d >= -14 ? static_cast<uint32_t>(d + 15) << 10 : d >= -24 ? 1u << (d + 24) : 0u;
    return h | h << 16;
}

template <int D>
__device__ void prompt_convert(const Attend8Params& p, const PromptJob& job, int seq, uint8_t* smem, uint64_t* bars, volatile int* flags) {
    using Smem = PromptSmem<D>;
    constexpr int kLoads = D / 32;               // 16-byte pieces of a lane and page
    constexpr uint32_t kColumn = 2048;           // K: bytes between 8-dim columns.  V: between groups of 8 tokens it is D * 16
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - 8;
    const uint32_t base = smem_u32(smem);
    const int32_t* table = p.tables + seq * p.table_stride;
    const int pages = pages_of_length(job.token_b);
    const int tok = lane & 15, half = lane >> 4;
    int* first_nan = reinterpret_cast<int*>(smem + Smem::kNan);
    StepDesc* descs = reinterpret_cast<StepDesc*>(smem + Smem::kDesc);
    bool bad = false;

    // Lane i < 8 knows page i of a tile: its block (asked for two tiles ahead) and its scales (one tile ahead, with the codes).
    auto ask_block = [&](int token0) {
        const int page = token0 / kPageTokens + (lane & 7);
        int block = -1;
        if (page < pages) {
            block = __ldg(table + page / p.pages_per_block);
            if (block < 0 || block >= p.num_blocks) {
                bad = true;
                block = block < 0 ? 0 : static_cast<int>(p.num_blocks - 1);
            }
        }
        return block;
    };
    uint4 k[2][kLoads], v[2][kLoads];
    float2 scales = make_float2(0.f, 0.f);
    auto page_at = [&](int token0, int i, int block) { return page_address<D>(p, token0 / kPageTokens + i, block, job.kvh); };
    auto ask_scales = [&](int token0, int block) {
        scales = block >= 0 ? __ldg(reinterpret_cast<const float2*>(page_at(token0, lane & 7, block) + cache8_scale_off(D))) : make_float2(0.f, 0.f);
    };
    auto ask_codes = [&](int token0, int block, bool values, uint4 (&x)[2][kLoads]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int b = __shfl_sync(0xffffffffu, block, 2 * warp + i);
            const uint8_t* at = b >= 0 ? page_at(token0, 2 * warp + i, b) + (values ? kPageTokens * D : 0) + tok * D + half * 16 : nullptr;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) x[i][j] = b >= 0 ? __ldg(reinterpret_cast<const uint4*>(at + j * 32)) : make_uint4(0, 0, 0, 0);
        }
    };
    int block = ask_block(job.token_a);
    ask_scales(job.token_a, block);
    ask_codes(job.token_a, block, false, k);
    ask_codes(job.token_a, block, true, v);
    block = ask_block(job.token_a + kTile);
    int step = 0;
    for (int token0 = job.token_a; token0 < job.token_b; token0 += kTile) {
        const bool last_tile = token0 + kTile >= job.token_b;
        const int ke = exponent_of_scale_bits(__float_as_uint(scales.x)), ve = exponent_of_scale_bits(__float_as_uint(scales.y));
        const bool here = token0 / kPageTokens + (lane & 7) < pages;
        const int k_ref = __reduce_max_sync(0xffffffffu, here ? ke : kMinExponent);
        uint32_t todo = 0xffu;                                              // pages that are still to come
        while (todo) {
            // The pages within 2^15 of the largest scale left; pages whose values are all zeros go with any.
            const bool open = todo >> (lane & 7) & 1, counts = here && ve > kMinExponent;
            const int v_ref = __reduce_max_sync(0xffffffffu, open && counts ? ve : kMinExponent);
            const uint32_t group = __ballot_sync(0xffffffffu, open && (!counts || ve >= v_ref - 15)) & 0xffu;
            todo &= ~group;
            const bool last = last_tile && !todo;
            const int s = step & 1;
            const uint32_t turn = (step >> 1 & 1) ^ 1;
            if (!mbar_wait_bounded(bars + kbKEmpty + s, turn)) flags[0] = 1;
            if (warp == 0 && lane == 0) {
                StepDesc& d = descs[step % kDescs];
                d.token0 = token0;
                d.mask = static_cast<int>(group);
                d.last = last;
                d.v_exp = v_ref;
                d.k_scale = exp2_int(k_ref);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int page = 2 * warp + i;
                const int d = max(__shfl_sync(0xffffffffu, ke, page) - k_ref, -126);
                const uint32_t f = half2_power(d);
                const uint32_t to = base + Smem::kK + s * Smem::kOperand + (page * kPageTokens + tok) * 16 + half * 2 * kColumn;
#pragma unroll
                for (int j = 0; j < kLoads; ++j) convert16<false>(k[i][j], f, d == 0, to + j * 4 * kColumn, kColumn);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) prompt_arrive(bars + kbKFull + s);
            if (!todo && !last) ask_codes(token0 + kTile, block, false, k);  // the next tile's, behind this one's last use

            if (!mbar_wait_bounded(bars + kbVEmpty + s, turn)) flags[0] = 1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int page = 2 * warp + i;
                const int d = max(min(__shfl_sync(0xffffffffu, ve, page) - v_ref, 0), -126);
                const bool in = group >> page & 1;
                const uint32_t f = in ? half2_power(d) : 0u;
                const int token = page * kPageTokens + tok;
                const uint32_t to = base + Smem::kV + s * Smem::kOperand + (token >> 3) * (D * 16) + (token & 7) * 16 + half * 256;
#pragma unroll
                for (int j = 0; j < kLoads; ++j) {
                    uint4 x = v[i][j];
                    uint32_t nan[4] = {x.x, x.y, x.z, x.w}, any = 0;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        nan[w] = ((nan[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                        any |= nan[w];
                    }
                    if (any) {
                        flags[1] = 1;
#pragma unroll
                        for (int w = 0; w < 4; ++w)
#pragma unroll
                            for (int b = 0; b < 4; ++b)
                                if (nan[w] >> (8 * b + 7) & 1) atomicMin(first_nan + (2 * j + half) * 16 + 4 * w + b, token0 + token);
                        x.x &= ~((nan[0] >> 7) * 0xffu);
                        x.y &= ~((nan[1] >> 7) * 0xffu);
                        x.z &= ~((nan[2] >> 7) * 0xffu);
                        x.w &= ~((nan[3] >> 7) * 0xffu);
                    }
                    convert16<true>(x, f, in && d == 0, to + j * 512, 128);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) prompt_arrive(bars + kbVFull + s);
            if (!todo && !last) {
                ask_codes(token0 + kTile, block, true, v);
                ask_scales(token0 + kTile, block);
                block = ask_block(token0 + 2 * kTile);
            }
            ++step;
            if (flags[0]) todo = 0;
        }
        if (flags[0]) break;
    }
    if (bad && p.status) atomicOr(p.status, TQ_STATUS_BAD_BLOCK);
}

template <int D>
__device__ void prompt_multiply(const PromptJob& job, uint8_t* smem, uint64_t* bars, volatile int* flags, uint32_t tmem) {
    using Smem = PromptSmem<D>;
    constexpr uint32_t kScores = prompt_idesc(kTile, 0), kOut = prompt_idesc(D, 1);
    const uint32_t base = smem_u32(smem);
    const StepDesc* descs = reinterpret_cast<const StepDesc*>(smem + Smem::kDesc);
    auto scores = [&](int q, int s) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            prompt_mma_ss(tmem + q * kTile, prompt_desc(base + Smem::kQ + q * Smem::kOperand + i * 4096, 2048, 128),
                          prompt_desc(base + Smem::kK + s * Smem::kOperand + i * 4096, 2048, 128), kScores, i ? 1u : 0u);
        prompt_commit(bars + kbSFull + q);
    };
    auto wait = [&](int bar, uint32_t parity) {
        if (!mbar_wait_bounded(bars + bar, parity)) flags[0] = 1;
        return flags[0] == 0;
    };
    if (!wait(kbKFull, 0)) return;
    prompt_fence_after();
    for (int q = 0; q < job.tiles; ++q) scores(q, 0);
    prompt_commit(bars + kbKEmpty);
    for (int step = 0;; ++step) {
        const int s = step & 1;
        const bool last = *const_cast<const volatile int*>(&descs[step % kDescs].last);
        if (!wait(kbVFull + s, step >> 1 & 1)) return;
        for (int q = 0; q < job.tiles; ++q) {
            if (!wait(kbPFull + q, step & 1)) return;
            prompt_fence_after();
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
                prompt_mma_ts(tmem + 2 * kTile + q * kTile, tmem + q * kTile + i * 8,
                              prompt_desc(base + Smem::kV + s * Smem::kOperand + i * 2 * (D * 16), D * 16, 128), kOut, step || i ? 1u : 0u);
            prompt_commit(bars + kbPvDone + q);
            if (q == job.tiles - 1) prompt_commit(bars + kbVEmpty + s);
            if (!last) {
                const int n = (step + 1) & 1;
                if (q == 0) {
                    if (!wait(kbKFull + n, (step + 1) >> 1 & 1)) return;
                    prompt_fence_after();
                }
                scores(q, n);
                if (q == job.tiles - 1) prompt_commit(bars + kbKEmpty + n);
            }
        }
        if (last) break;
    }
}

template <int D>
__device__ void prompt_softmax(const Attend8Params& p, const PromptJob& job, int split, uint8_t* smem, uint64_t* bars, volatile int* flags, uint32_t tmem,
                               bool bf16, float row_scale) {
    using Smem = PromptSmem<D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = warp >> 2;
    const int row = job.r0 + q * kTile + (warp & 3) * 32 + lane;
    const int limit = job.len - job.nq + min(row, job.nrows - 1) / p.group + 1;
    const int warp_limit = __reduce_min_sync(0xffffffffu, limit);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + q * kTile, o_at = tmem + lanes + 2 * kTile + q * kTile;
    const StepDesc* descs = reinterpret_cast<const StepDesc*>(smem + Smem::kDesc);
    float m = kNothing, u = kNothing, l = 0.f;
    bool ok = true;
    if (job.token_a < job.token_b) {
        for (int step = 0;; ++step) {
            if (!mbar_wait_bounded(bars + kbSFull + q, step & 1)) flags[0] = 1;
            if (flags[0]) {
                ok = false;
                break;
            }
            prompt_fence_after();
            const StepDesc d = descs[step % kDescs];
            const float c = fmaxf(row_scale * d.k_scale, 1e-38f), ev = static_cast<float>(d.v_exp);
            const bool masked = d.mask != 0xff || d.token0 + kTile > warp_limit;
            const int visible = limit - d.token0;
            float most = -__uint_as_float(0x7f800000u);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                uint32_t x[32];
                prompt_ld32(s_at + 32 * h, x);
                prompt_wait_ld();
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * h + i >= visible || !(d.mask >> (2 * h + (i >> 4)) & 1)) x[i] = 0xff800000u;
                }
                float a = most, b = most;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    a = fmaxf(fmaxf(a, __uint_as_float(x[i])), __uint_as_float(x[i + 1]));
                    b = fmaxf(fmaxf(b, __uint_as_float(x[i + 2])), __uint_as_float(x[i + 3]));
                }
                most = fmaxf(a, b);
            }
            most *= c;
            if (__any_sync(0xffffffffu, most > fminf(m, u - ev) + kLazy)) {
                const float m1 = fmaxf(m, most), u1 = fmaxf(u, most + ev);
                l *= ex2(m - m1);
                const float down = ex2(u - u1);
                m = m1;
                u = u1;
                if (step) {
                    // O is whole when the product of the step before is done
                    if (!mbar_wait_bounded(bars + kbPvDone + q, (step - 1) & 1)) flags[0] = 1;
                    prompt_fence_after();
#pragma unroll
                    for (int h = 0; h < D / 32; ++h) {
                        uint32_t x[32];
                        prompt_ld32(o_at + 32 * h, x);
                        prompt_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * down);
                        prompt_st32(o_at + 32 * h, x);
                    }
                }
            }
            const float shift = ev + kHeadroom - u;
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                uint32_t x[32], w[16];
                prompt_ld32(s_at + 32 * h, x);
                prompt_wait_ld();
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * h + i >= visible || !(d.mask >> (2 * h + (i >> 4)) & 1)) x[i] = 0xff800000u;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float a = ex2(fmaf(__uint_as_float(x[2 * i]), c, shift)), b = ex2(fmaf(__uint_as_float(x[2 * i + 1]), c, shift));
                    sum0 += a;
                    sum1 += b;
                    w[i] = pack_half2(a, b);
                }
                prompt_st16(s_at + 16 * h, w);
            }
            l = fmaf(sum0 + sum1, ex2(u - ev - kHeadroom - m), l);
            prompt_wait_st();
            prompt_fence_before();
            __syncwarp();
            if (lane == 0) prompt_arrive(bars + kbPFull + q);
            if (d.last) {
                if (!mbar_wait_bounded(bars + kbPvDone + q, step & 1)) flags[0] = 1;
                ok = flags[0] == 0;
                prompt_fence_after();
                break;
            }
        }
    }
    // The row's values: in units of the weights' reference, divided by their sum where this CTA saw all of them.
    const bool whole = p.chunks == 1;
    const bool store = ok && row < job.nrows;
    const int token = row / p.group, head = job.kvh * p.group + row - token * p.group;
    const int64_t at = static_cast<int64_t>(job.first_row + token) * p.q_heads + head;
    float f = l == 0.f ? 0.f : ex2(u - m - kHeadroom);
    if (whole && l != 0.f) f /= l;
    const bool nothing = job.token_a >= job.token_b || l == 0.f;
    const int* first_nan = reinterpret_cast<const int*>(smem + Smem::kNan);
#pragma unroll
    for (int h = 0; h < D / 32; ++h) {
        uint32_t x[32];
        if (job.token_a < job.token_b && ok) {
            prompt_ld32(o_at + 32 * h, x);
            prompt_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = nothing ? 0u : __float_as_uint(__uint_as_float(x[i]) * f);
        if (flags[1]) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (first_nan[32 * h + i] < limit) x[i] = 0x7fffffffu;
        }
        if (!store) continue;
        if (whole) {
            uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at * D + 32 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack_out(__uint_as_float(x[8 * i + 2 * j]), __uint_as_float(x[8 * i + 2 * j + 1]), bf16);
                to[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            float2* to = reinterpret_cast<float2*>(p.partials + (at * p.chunks + split) * (D + 2) + 32 * h);
#pragma unroll
            for (int i = 0; i < 16; ++i) to[i] = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
        }
    }
    if (store && !whole) *reinterpret_cast<float2*>(p.partials + (at * p.chunks + split) * (D + 2) + D) = make_float2(m, l);
}

// Queries of a tile as K-major A operand, thread = row; returns the factor of its scores in units of log2.
template <int D>
__device__ float prompt_queries(const Attend8Params& p, const PromptJob& job, uint8_t* smem, bool bf16) {
    using Smem = PromptSmem<D>;
    const int q = threadIdx.x / kTile, r = threadIdx.x % kTile, row = job.r0 + threadIdx.x;
    uint32_t x[D / 2];
    if (row < job.nrows) {
        const int token = row / p.group, head = job.kvh * p.group + row - token * p.group;
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(job.first_row + token) * p.q_heads + head) * D);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const uint4 w = __ldg(from + i);
            x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < D / 2; ++i) x[i] = 0;
    }
    float row_scale = fabsf(p.scale_log2);
    if (bf16) {      // into the range of fp16 by a power of two, as in load_queries
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < D / 2; ++i) most = max(most, max(x[i] & 0x7fffu, x[i] >> 16 & 0x7fffu));
        const int e = min(max(static_cast<int>(most >> 7) - 127, -120), 120);
        const float down = exp2_int(-e);
#pragma unroll
        for (int i = 0; i < D / 2; ++i) x[i] = pack_half2(__uint_as_float(x[i] << 16) * down, __uint_as_float(x[i] & 0xffff0000u) * down);
        row_scale *= exp2_int(e);
    }
    const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    const uint32_t to = smem_u32(smem) + Smem::kQ + q * Smem::kOperand + r * 16;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) sts16(to + i * 2048, x[4 * i] ^ sign, x[4 * i + 1] ^ sign, x[4 * i + 2] ^ sign, x[4 * i + 3] ^ sign);
    return row_scale;
}

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1) attend8_prompt_kernel(const Attend8Params p, int bf16) {
    using Smem = PromptSmem<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
    volatile int* flags = reinterpret_cast<volatile int*>(smem + Smem::kFlags);
    const int tid = threadIdx.x, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + kbKFull + i, 4);
            mbar_init(bars + kbKEmpty + i, 1);
            mbar_init(bars + kbVFull + i, 4);
            mbar_init(bars + kbVEmpty + i, 1);
            mbar_init(bars + kbSFull + i, 1);
            mbar_init(bars + kbPFull + i, 4);
            mbar_init(bars + kbPvDone + i, 1);
        }
        flags[0] = flags[1] = 0;
        fence_barrier_init();
    }
    for (int i = tid; i < D; i += kPromptThreads) reinterpret_cast<int*>(smem + Smem::kNan)[i] = INT32_MAX;
    pdl_wait();
    pdl_release();

    // splits of one block of rows side by side, then the KV heads, then blocks of rows from the last one, which sees the most, down
    int rest = blockIdx.x;
    const int split = rest % p.chunks;
    rest /= p.chunks;
    PromptJob job;
    job.kvh = rest % p.kv_heads;
    rest /= p.kv_heads;
    const int seq = rest % p.seqs, block = p.tiles - 1 - rest / p.seqs;
    if (p.zero_tail && blockIdx.x == 0) {
        const int64_t row = static_cast<int64_t>(p.q_heads) * D, used = p.starts ? min(max(p.starts[p.seqs], 0), p.rows) : p.seqs;
        for (int64_t i = used * row + tid; i < p.rows * row; i += kPromptThreads) static_cast<uint16_t*>(p.out)[i] = 0;
    }
    const bool too_many = rows_of(p, seq, job.first_row, job.nq);
    job.nrows = job.nq * p.group;
    job.r0 = block * 2 * kTile;
    job.len = p.seq_lens[seq];
    const bool too_long = pages_of_length(job.len) > p.max_pages;
    if (too_long) job.len = p.max_pages * kPageTokens;
    if ((too_long || too_many) && p.status && tid == 0 && split == 0 && block == 0 && job.kvh == 0)
        atomicOr(p.status, (too_long ? TQ_STATUS_BAD_BLOCK : 0) | (too_many ? TQ_STATUS_TOO_LONG : 0));
    if (job.r0 >= job.nrows) return;
    job.tiles = job.nrows - job.r0 > kTile ? 2 : 1;
    const int most = max(job.len - job.nq + min(job.r0 + 2 * kTile - 1, job.nrows - 1) / p.group + 1, 0);
    const int steps = (most + kTile - 1) / kTile, each = (steps + p.chunks - 1) / p.chunks;
    job.token_a = min(split * each * kTile, most);
    job.token_b = min((split + 1) * each * kTile, most);

    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem) + Smem::kTmemSlot), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    float row_scale = 0.f;
    if (warp < 4 * job.tiles) {
        row_scale = prompt_queries<D>(p, job, smem, bf16 != 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    prompt_fence_before();
    __syncthreads();
    prompt_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + Smem::kTmemSlot);
    if (warp < 8) {
        if (warp < 4 * job.tiles) prompt_softmax<D>(p, job, split, smem, bars, flags, tmem, bf16 != 0, row_scale);
    } else if (warp < 12) {
        prompt_convert<D>(p, job, seq, smem, bars, flags);
    } else if ((tid & 31) == 0 && job.token_a < job.token_b) {
        prompt_multiply<D>(job, smem, bars, flags, tmem);
    }
    __syncwarp();
    if (flags[0] && p.status && (tid & 31) == 0) atomicOr(p.status, TQ_STATUS_TIMEOUT);
    prompt_fence_before();
    __syncthreads();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace
}  // namespace tq
