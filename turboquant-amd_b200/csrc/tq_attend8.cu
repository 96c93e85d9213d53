// Attention over the 8-bit paged cache (tq_cache8.cuh): queries of one token per sequence, of a few, or of a chunk of a prompt whose
// keys are in the cache already.
//
// For a query row (token j of n in a sequence of `len` tokens, head h) with KV head h / G:
//   s_k = sm_scale * <q, K_k> * kscale(page of k)      for k < len - n + j + 1
//   out = sum_k 2^(s_k - m) vscale(page of k) V_k / sum_k 2^(s_k - m)      (s in units of log2)
//
// Bound: HBM, the 2 D + 2 bytes of a cached token and head.  8 query rows take D / 8 products (m16n8k16) a page of 16 tokens; with D = 128 the persistent
// kernel issues 359 warp instructions a page in all, at half of the issue slots.
#include "tq_cache8.cuh"

namespace tq {
namespace {

struct Attend8Params {
    void* out;
    const void* q;
    const uint8_t* cache;
    const int32_t* tables;
    const int32_t* seq_lens;
    const int32_t* starts;          // [seqs + 1], null: row i is sequence i's only one
    float* partials;
    int32_t* status;
    int64_t num_blocks, table_stride;
    float scale_log2;
    int rows, seqs, q_heads, kv_heads, group, pages_per_block, max_pages, max_queries, tiles, chunks, zero_rest;
    int small_rows;                 // not 0: sequences of at most so many query rows have one kernel, the others another one
};

constexpr float kNothing = -3e38f;      // reference of a row that has seen no token: below every score, and finite, so that differences are numbers
constexpr float kLazy = 8.f;            // a score may pass the reference by so much before it is raised
constexpr float kHeadroom = 7.f;        // weights are multiplied by 2^7: at most 2^15 in fp16, full precision down to 2^-21 of the largest

// What one warp holds while it walks over pages of a sequence, for 8 * NT query rows against one KV head.
//
// Scores: m16n8k16 products with 16 tokens as M and query rows as N.  A lane (g = lane / 4, t = lane % 4) reads 16-byte pieces t (and t + 4) of
// tokens g and g + 8: four dims are one operand register pair, with the query laid out alike, so the codes need no shuffling at all.
// Values: V^T as the A operand (dims as M).  A lane reads dims D/8 * g .. of tokens 2t, 2t + 1, 2t + 8, 2t + 9 - whole 128-byte
// rows - and a byte permute pairs the tokens.  Weights go from accumulator to operand layout by two movmatrix.
template <int D, int NT>
struct Rows {
    static constexpr int kSteps = D / 16;      // products of a page's scores, and m-tiles of its values
    uint32_t q[NT][kSteps][2];
    float scale[NT][2];                        // of the two columns of this lane
    float m[NT][2], u[NT][2], l[NT][2];        // references of weights and of weights * vscale, denominators of this lane
    float o[kSteps][NT][4];
    int limit[NT][2];                          // tokens that the column sees
    int min_limit, max_limit;
};

template <int D>
struct Page {
    uint4 k[2][D / 64];
    uint32_t v[4][D / 32];
    float2 scales;
};

template <int D>
__device__ __forceinline__ const uint8_t* page_address(const Attend8Params& p, int page, int block, int kvh) {
    return p.cache + ((static_cast<int64_t>(block) * p.kv_heads + kvh) * p.pages_per_block + page % p.pages_per_block) *
                         static_cast<int64_t>(cache8_page_bytes(D));
}

template <int D>
__device__ __forceinline__ void load_keys(Page<D>& x, const uint8_t* base, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) x.k[r][c] = __ldg(reinterpret_cast<const uint4*>(base + (g + 8 * r) * D + 64 * c + 16 * t));
    x.scales = __ldg(reinterpret_cast<const float2*>(base + cache8_scale_off(D)));
}

template <int D>
__device__ __forceinline__ void load_values(Page<D>& x, const uint8_t* base, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint8_t* at = base + kPageTokens * D + (2 * t + (i & 1) + 8 * (i >> 1)) * D + D / 8 * g;
        if constexpr (D == 128) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(at));
            x.v[i][0] = w.x; x.v[i][1] = w.y; x.v[i][2] = w.z; x.v[i][3] = w.w;
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(at));
            x.v[i][0] = w.x; x.v[i][1] = w.y;
        }
    }
}

// Query rows r0 .. r0 + 8 NT of a sequence as B operands.  fp16 queries are used as they are; bf16 ones are brought into the range of
// fp16 by a power of two for each row, which costs no bit of values within 2^-14 of the row's largest.
template <int D, int NT>
struct QueryWords {
    uint32_t x[NT][D / 64][8];
};

template <int D, int NT>
__device__ __forceinline__ void ask_queries(QueryWords<D, NT>& w, const Attend8Params& p, int first_row, int kvh, int r0, int nrows, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = r0 + 8 * n + g;
        uint32_t(&x)[D / 64][8] = w.x[n];
        if (r < nrows) {
            const int token = r / p.group, head = kvh * p.group + r - token * p.group;
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(first_row + token) * p.q_heads + head) * D + 16 * t;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const uint4 a = __ldg(reinterpret_cast<const uint4*>(src + 64 * c)), b = __ldg(reinterpret_cast<const uint4*>(src + 64 * c + 8));
                x[c][0] = a.x; x[c][1] = a.y; x[c][2] = a.z; x[c][3] = a.w;
                x[c][4] = b.x; x[c][5] = b.y; x[c][6] = b.z; x[c][7] = b.w;
            }
        } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[c][i] = 0;
        }
    }
}

template <int D, int NT, bool BF16>
__device__ __forceinline__ void set_queries(Rows<D, NT>& w, QueryWords<D, NT>& words, const Attend8Params& p, int r0, int nrows, int len, int nq, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        uint32_t(&x)[D / 64][8] = words.x[n];
        float row_scale = fabsf(p.scale_log2);
        if (p.scale_log2 < 0.f) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[c][i] ^= 0x80008000u;
        }
        if constexpr (BF16) {
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) most = max(most, max(x[c][i] & 0x7fffu, x[c][i] >> 16 & 0x7fffu));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e = min(max(static_cast<int>(most >> 7) - 127, -120), 120);
            const float down = exp2_int(-e);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[c][i] = pack_half2(__uint_as_float(x[c][i] << 16) * down, __uint_as_float(x[c][i] & 0xffff0000u) * down);
            row_scale *= exp2_int(e);
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w.q[n][4 * c + i][0] = x[c][2 * i];
                w.q[n][4 * c + i][1] = x[c][2 * i + 1];
            }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            w.scale[n][j] = __shfl_sync(0xffffffffu, row_scale, (2 * t + j) * 4);
            const int row = r0 + 8 * n + 2 * t + j;
            w.limit[n][j] = len - nq + min(row, nrows - 1) / p.group + 1;
            w.m[n][j] = w.u[n][j] = kNothing;
            w.l[n][j] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < Rows<D, NT>::kSteps; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) w.o[i][n][j] = 0.f;
    w.min_limit = len - nq + r0 / p.group + 1;
    w.max_limit = len - nq + min(r0 + 8 * NT - 1, nrows - 1) / p.group + 1;
}

template <int D, int NT, bool BF16>
__device__ __forceinline__ void load_queries(Rows<D, NT>& w, const Attend8Params& p, int first_row, int kvh, int r0, int nrows, int len, int nq, int lane) {
    QueryWords<D, NT> words;
    ask_queries<D, NT>(words, p, first_row, kvh, r0, nrows, lane);
    set_queries<D, NT, BF16>(w, words, p, r0, nrows, len, nq, lane);
}

template <int D, int NT>
__device__ __forceinline__ void page_scores(float (&s)[NT][4], const Rows<D, NT>& w, const Page<D>& x) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        const uint32_t a[4] = {x.k[0][c].x, x.k[0][c].y, x.k[0][c].z, x.k[0][c].w}, b[4] = {x.k[1][c].x, x.k[1][c].y, x.k[1][c].z, x.k[1][c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = e4m3x2_to_half2(a[i] & 0xffffu), a1 = e4m3x2_to_half2(b[i] & 0xffffu);
            const uint32_t a2 = e4m3x2_to_half2(a[i] >> 16), a3 = e4m3x2_to_half2(b[i] >> 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(s[n], a0, a1, a2, a3, w.q[n][4 * c + i][0], w.q[n][4 * c + i][1]);
        }
    }
}

// Adds weights * V.  Tokens of the page from `visible` on count as zeros, whatever their codes say.
template <int D, int NT, bool CUT>
__device__ __forceinline__ void page_values(float (&o)[D / 16][NT][4], const Page<D>& x, const uint32_t (&weights)[NT][2], int visible, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = !CUT || 2 * t + (j & 1) + 8 * (j >> 1) < visible ? x.v[j][i] : 0u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t lo = prmt(v[0], v[1], h ? 0x7362 : 0x5140), hi = prmt(v[2], v[3], h ? 0x7362 : 0x5140);
            const uint32_t a0 = e4m3x2_to_half2(lo & 0xffffu), a1 = e4m3x2_to_half2(lo >> 16);
            const uint32_t a2 = e4m3x2_to_half2(hi & 0xffffu), a3 = e4m3x2_to_half2(hi >> 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(o[2 * i + h][n], a0, a1, a2, a3, weights[n][0], weights[n][1]);
        }
    }
}

template <int D>
__device__ __forceinline__ bool has_nan(const Page<D>& x, int from, int lane) {
    const int t = lane & 3;
    uint32_t found = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint32_t full = (x.v[j][i] & 0x7f7f7f7fu) + 0x01010101u;      // bit 7 of a byte: it is 0x7f
            if (2 * t + (j & 1) + 8 * (j >> 1) >= from) found |= full & 0x80808080u;
        }
    return __any_sync(0xffffffffu, found != 0);
}

// A page's value scale may lie so many powers of two below the reference: fp16 then holds weights down to 2^-30 of the largest, and what is lost is
// 2^-30 of the values for each token.  (Two, one of which the reference's rounding up may take, and what rounding makes of the difference.)
constexpr float kLossless = 2.01f;

// One page.  The softmax keeps two references per column: m for the denominators and u, a whole number, which includes the value scale 2^ev of the page, for
// the products, whose fp16 weights then use their range whatever the pages' scales are.  Both are raised only where a score passes
// them by 2^8: most pages need two votes and no shuffles.
template <int D, int NT>
__device__ __forceinline__ void page_weights(Rows<D, NT>& w, float (&s)[NT][4], float2 scales, int page, uint32_t (&weights)[NT][2]) {
    const int g = (threadIdx.x & 31) >> 2;
    const float ev = static_cast<float>(static_cast<int>(__float_as_uint(scales.y) >> 23 & 0xffu) - 127);
    float c[NT][2];         // positive: the sign of sm_scale is in the query
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) c[n][j] = w.scale[n][j] * scales.x;
    if (page * kPageTokens + kPageTokens > w.min_limit) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[n][j] = page * kPageTokens + g + 8 * (j >> 1) >= w.limit[n][j & 1] ? -__uint_as_float(0x7f800000u) : s[n][j] * c[n][j & 1];
            c[n][0] = c[n][1] = 1.f;
        }
    }
    bool over = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) over |= fmaxf(s[n][j], s[n][j + 2]) * c[n][j] > fminf(w.m[n][j], w.u[n][j] - ev) + kLazy;
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float most = fmaxf(s[n][j], s[n][j + 2]) * c[n][j];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float m = fmaxf(w.m[n][j], most), u = fmaxf(w.u[n][j], ceilf(most + ev));
                w.l[n][j] *= ex2(w.m[n][j] - m);
                const float down = exp2_int(static_cast<int>(fmaxf(w.u[n][j] - u, -127.f)));        // exact; 2^-127 is zero
#pragma unroll
                for (int i = 0; i < Rows<D, NT>::kSteps; ++i) {
                    w.o[i][n][j] *= down;
                    w.o[i][n][j + 2] *= down;
                }
                w.m[n][j] = m;
                w.u[n][j] = u;
            }
    }
    bool apart = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) apart |= w.u[n][j] - ev - w.m[n][j] > kLossless;
    // Where the page's values are 2^up below the reference, fp16 would lose every weight below 2^(up - 32) of the largest: there may be many,
    // they count for the denominator, and for the output where the large values are zeros.  So u is lowered, and the sums are multiplied by
    // as much, for which fp32 has room up to 2^100.  Where that does not suffice, the page's weights are for the denominator alone,
    // in units of m, and add nothing to sums of that size.
    uint32_t far = 0;                   // bit 2 n + j
    if (__any_sync(0xffffffffu, apart)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float big = 0.f;
#pragma unroll
                for (int i = 0; i < Rows<D, NT>::kSteps; ++i) big = fmaxf(big, fmaxf(fabsf(w.o[i][n][j]), fabsf(w.o[i][n][j + 2])));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                const int room = min(100 + 127 - static_cast<int>(__float_as_uint(big) >> 23), 120);
                int d = static_cast<int>(fmaxf(floorf(w.u[n][j] - ev - w.m[n][j]), 0.f));
                if (d > room) {
                    far |= 1u << (2 * n + j);
                    d = 0;
                }
                const float lift = exp2_int(d);
                w.u[n][j] -= static_cast<float>(d);
#pragma unroll
                for (int i = 0; i < Rows<D, NT>::kSteps; ++i) {
                    w.o[i][n][j] *= lift;
                    w.o[i][n][j + 2] *= lift;
                }
            }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float shift[2], unit[2], e[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            shift[j] = ev + kHeadroom - w.u[n][j];
            unit[j] = -shift[j] - w.m[n][j];
            if (far >> (2 * n + j) & 1) {
                shift[j] = kHeadroom - w.m[n][j];
                unit[j] = -kHeadroom;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = ex2(fmaf(s[n][j], c[n][j & 1], shift[j & 1]));
        // The denominator sums the weights as they are rounded for the product, so that a rounding common to both cancels: a token that takes
        // nearly all is then exact.
        uint32_t lo = pack_half2(e[0], e[1]), hi = pack_half2(e[2], e[3]);
        const float2 a = unpack_half2(lo), b = unpack_half2(hi);
        w.l[n][0] = fmaf(a.x + b.x, ex2(unit[0]), w.l[n][0]);
        w.l[n][1] = fmaf(a.y + b.y, ex2(unit[1]), w.l[n][1]);
        if (far) {
            const uint32_t keep = (far >> (2 * n) & 1 ? 0u : 0xffffu) | (far >> (2 * n + 1) & 1 ? 0u : 0xffff0000u);
            lo &= keep;
            hi &= keep;
        }
        weights[n][0] = movmatrix_trans(lo);        // tokens 2t, 2t + 1 of column g
        weights[n][1] = movmatrix_trans(hi);
    }
}

template <int D, int NT>
__device__ __forceinline__ void page_products(Rows<D, NT>& w, const Page<D>& x, const uint32_t (&weights)[NT][2], int page, int lane) {
    const int first = page * kPageTokens;
    if (first + kPageTokens <= w.min_limit) {
        page_values<D, NT, false>(w.o, x, weights, kPageTokens, lane);
        return;
    }
    const int most = min(w.max_limit - first, kPageTokens), least = max(min(w.min_limit - first, kPageTokens), 0);
    if (most <= least || !has_nan<D>(x, least, lane)) {
        page_values<D, NT, true>(w.o, x, weights, most, lane);
        return;
    }
    // A NaN that some columns see and others do not: 0 * NaN would reach the latter.  It counts as zero in the product, and a second
    // one, of ones where NaN stand with ones where a column sees a token, says where it belongs.
    const int g = lane >> 2, t = lane & 3;
    Page<D> clean, marks;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint32_t nan = ((x.v[j][i] & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u;
            clean.v[j][i] = x.v[j][i] & ~(nan * 0xffu);
            marks.v[j][i] = nan * 0x38u;               // 1.0 in e4m3
        }
    page_values<D, NT, true>(w.o, clean, weights, most, lane);
    uint32_t sees[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        // the limit of column g of this tile is held by the lanes whose t is g / 2
        const int lo = __shfl_sync(0xffffffffu, w.limit[n][0], g >> 1), hi = __shfl_sync(0xffffffffu, w.limit[n][1], g >> 1);
        const int mine = (g & 1 ? hi : lo) - first;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            sees[n][h] = (2 * t + 8 * h < mine ? 0x3c00u : 0u) | (2 * t + 1 + 8 * h < mine ? 0x3c000000u : 0u);
    }
    float found[D / 16][NT][4] = {};
    page_values<D, NT, true>(found, marks, sees, most, lane);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (found[i][n][j] > 0.f) w.o[i][n][j] = __uint_as_float(0x7fffffffu);
}

constexpr int kMaxCluster = 8;

__device__ __forceinline__ uint32_t cluster_address(uint32_t at, int cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(cta));
    return r;
}
__device__ __forceinline__ float2 load_cluster2(uint32_t at) {
    float2 x;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
    return x;
}

__device__ __forceinline__ uint32_t pack_out(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    return pack_half2(a, b);
}

// A query row's output from its D / 32 sums of each lane.
template <int D, bool BF16>
__device__ __forceinline__ void store_row(const Attend8Params& p, int first_row, int kvh, int row, const float (&o)[D / 32], float l, int lane) {
    const int token = row / p.group, head = kvh * p.group + row - token * p.group;
    uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + (static_cast<int64_t>(first_row + token) * p.q_heads + head) * D) + lane * (D / 64);
    const float f = 1.f / l;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) to[i] = l == 0.f ? 0u : pack_out(o[2 * i] * f, o[2 * i + 1] * f, BF16);
}

__device__ __forceinline__ void store_out(void* out, int64_t at, float x, bool bf16) {
    if (bf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(x);
    else static_cast<__half*>(out)[at] = __float2half_rn(x);
}

// The rows of a sequence, inside the tensors whatever `starts` says; returns how many more it has than the launch is sized for, which are left out.
__device__ __forceinline__ int rows_of(const Attend8Params& p, int seq, int& first_row, int& nq) {
    first_row = seq;
    nq = 1;
    if (!p.starts) return 0;
    first_row = min(max(p.starts[seq], 0), p.rows);
    const int n = max(min(p.starts[seq + 1], p.rows) - first_row, 0);
    nq = min(n, p.max_queries);
    return n - nq;
}

// A block's threads write zeros to rows a .. b.
template <int D>
__device__ __forceinline__ void zero_rows(const Attend8Params& p, int a, int b) {
    const int64_t row = static_cast<int64_t>(p.q_heads) * D / 8;
    uint4* out = static_cast<uint4*>(p.out);
    for (int64_t i = a * row + threadIdx.x; i < b * row; i += blockDim.x) out[i] = make_uint4(0, 0, 0, 0);
}

// Rows before the first sequence and behind the last one.
template <int D>
__device__ __forceinline__ void zero_ends(const Attend8Params& p) {
    if (p.starts) zero_rows<D>(p, 0, min(max(p.starts[0], 0), p.rows));
    zero_rows<D>(p, p.starts ? min(max(p.starts[p.seqs], 0), p.rows) : p.seqs, p.rows);
}

// Launches of few pages: a cluster of CTAs for each item (sequence, KV head, tile of 8 NT query rows), pages dealt out to the warps in
// turn, so that which pages a warp has does not depend on the length, and length, block table and query are asked for together.  Parts are
// joined in shared memory, those of the CTAs through distributed shared memory: a second kernel for that took as long as
// the first (1 x 4096 tokens, 64 / 8 heads: 13.1 us with it, 7.8 without).
__host__ __device__ constexpr int few_smem(int d, int nt, int warps) { return warps * 8 * nt * (d + 2) * 4 + 8 * nt * (d + 2) * 4; }

template <int D, int NT, bool BF16, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 4 && NT == 1 ? 4 : 1) attend8_few_kernel(const Attend8Params p) {
    constexpr int COLS = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    float* part_o = reinterpret_cast<float*>(smem);                 // [WARPS][COLS][D]
    float* part_s = part_o + WARPS * COLS * D;                      // [WARPS][COLS][2]: reference, denominator
    float* own_o = part_s + WARPS * COLS * 2;                       // [COLS][D], this CTA's
    float* own_s = own_o + COLS * D;                                // [COLS][2]
    pdl_wait();
    pdl_release_if_small();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    int rest = blockIdx.x;
    const int part = rest % p.chunks;                               // of the item: CTA of the cluster
    rest /= p.chunks;
    const int tile = rest % p.tiles;
    rest /= p.tiles;
    const int kvh = rest % p.kv_heads, seq = rest / p.kv_heads;
    const int32_t* table = p.tables + seq * p.table_stride;
    const int first = part * WARPS + warp, stride = p.chunks * WARPS;
    bool bad = false;
    auto ask = [&](int page) { return page < p.max_pages ? __ldg(table + page / p.pages_per_block) : 0; };
    int block = ask(first);
    if (p.zero_rest && blockIdx.x == 0) zero_ends<D>(p);
    int first_row, nq;
    const int left_out = rows_of(p, seq, first_row, nq);
    const int nrows = nq * p.group, r0 = tile * COLS;
    if (r0 >= nrows) return;                                        // the whole cluster
    if (left_out && p.zero_rest && part == 0 && tile == 0 && kvh == 0) zero_rows<D>(p, first_row + nq, first_row + nq + left_out);
    int len = p.seq_lens[seq];
    QueryWords<D, NT> words;
    ask_queries<D, NT>(words, p, first_row, kvh, r0, nrows, lane);
    const bool too_long = pages_of_length(len) > p.max_pages;
    if (too_long) len = p.max_pages * kPageTokens;
    if ((too_long || left_out) && p.status && tid == 0 && part == 0 && tile == 0 && kvh == 0)
        atomicOr(p.status, (too_long ? TQ_STATUS_BAD_BLOCK : 0) | (left_out ? TQ_STATUS_TOO_LONG : 0));
    const int most = len - nq + min(r0 + COLS - 1, nrows - 1) / p.group + 1, pages = pages_of_length(most);
    auto address = [&](int page) {
        if (block < 0 || block >= p.num_blocks) {
            bad = true;
            block = block < 0 ? 0 : static_cast<int>(p.num_blocks - 1);
        }
        return page_address<D>(p, page, block, kvh);
    };
    Page<D> x;
    if (first < pages) {
        const uint8_t* base = address(first);
        load_keys<D>(x, base, lane);
        load_values<D>(x, base, lane);
        block = ask(first + stride);
    }
    Rows<D, NT> w;
    set_queries<D, NT, BF16>(w, words, p, r0, nrows, len, nq, lane);
#pragma unroll 1
    for (int page = first; page < pages; page += stride) {
        const bool more = page + stride < pages;
        const uint8_t* next = more ? address(page + stride) : nullptr;
        float s[NT][4];
        uint32_t weights[NT][2];
        page_scores<D, NT>(s, w, x);
        const float2 scales = x.scales;
        if (more) load_keys<D>(x, next, lane);
        page_weights<D, NT>(w, s, scales, page, weights);
        page_products<D, NT>(w, x, weights, page, lane);
        if (more) {
            load_values<D>(x, next, lane);
            block = ask(page + 2 * stride);
        }
    }
    if (bad && p.status) atomicOr(p.status, TQ_STATUS_BAD_BLOCK);

    // The warps' parts, with the values in units of the weights' reference.
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float l = w.l[n][j];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const int col = 8 * n + 2 * t + j;
            const float up = ex2(w.u[n][j] - w.m[n][j] - kHeadroom);
            float* at = part_o + (warp * COLS + col) * D + D / 8 * g;
#pragma unroll
            for (int i = 0; i < D / 16; i += 2)
                *reinterpret_cast<float4*>(at + 2 * i) =
                    make_float4(w.o[i][n][j] * up, w.o[i][n][j + 2] * up, w.o[i + 1][n][j] * up, w.o[i + 1][n][j + 2] * up);
            if (g == 0) *reinterpret_cast<float2*>(part_s + (warp * COLS + col) * 2) = make_float2(w.m[n][j], l);
        }
    __syncthreads();
    // A warp joins the parts of one row at a time: lane k < WARPS knows warp k's statistics, a lane sums D / 32 dims.
    for (int col = warp; col < COLS; col += WARPS) {
        const int row = r0 + col;
        const float2 stat = lane < WARPS ? *reinterpret_cast<const float2*>(part_s + (lane * COLS + col) * 2) : make_float2(kNothing, 0.f);
        float m = stat.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float f = ex2(stat.x - m);
        float l = f * stat.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        float o[D / 32] = {};
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const float* at = part_o + (k * COLS + col) * D + lane * (D / 32);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] += fk * at[i];
        }
        if (p.chunks == 1) {
            if (row < nrows) store_row<D, BF16>(p, first_row, kvh, row, o, l, lane);
        } else {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) own_o[col * D + lane * (D / 32) + i] = o[i];
            if (lane == 0) {
                own_s[col * 2] = m;
                own_s[col * 2 + 1] = l;
            }
        }
    }
    if (p.chunks == 1) return;
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    // Rows are dealt out to the CTAs; lane k knows CTA k's statistics.
    for (int col = part + p.chunks * warp; col < COLS; col += p.chunks * WARPS) {
        const int row = r0 + col;
        if (row >= nrows) continue;
        float2 stat = load_cluster2(cluster_address(smem_u32(own_s + col * 2), lane < p.chunks ? lane : 0));
        float from[kMaxCluster][D / 32];
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            const uint32_t at = cluster_address(smem_u32(own_o + col * D + lane * (D / 32)), k < p.chunks ? k : 0);
#pragma unroll
            for (int i = 0; i < D / 32; i += 2) {
                const float2 x2 = load_cluster2(at + 4 * i);
                from[k][i] = x2.x;
                from[k][i + 1] = x2.y;
            }
        }
        if (lane >= p.chunks) stat = make_float2(kNothing, 0.f);
        float m = stat.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float f = lane < p.chunks ? ex2(stat.x - m) : 0.f;
        float l = f * stat.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        float o[D / 32] = {};
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            if (k < p.chunks) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] += fk * from[k][i];
            }
        }
        store_row<D, BF16>(p, first_row, kvh, row, o, l, lane);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // nobody's memory is read any more
}

// One warp per query row joins the parts of prompt attention whose keys were shared out.
template <int D>
__global__ void __launch_bounds__(128) attend8_merge_kernel(const Attend8Params p, int bf16) {
    pdl_release();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (at >= static_cast<int64_t>(p.rows) * p.q_heads) return;
    const int row = static_cast<int>(at / p.q_heads);
    int seq = p.starts ? 0 : row, end = p.seqs;                     // the last sequence that begins at or before the row
    while (p.starts && end - seq > 1) {
        const int mid = (seq + end) >> 1;
        if (p.starts[mid] <= row) seq = mid;
        else end = mid;
    }
    if (seq >= p.seqs) return;
    int first_row, nq;
    rows_of(p, seq, first_row, nq);
    if (row < first_row || row - first_row >= nq || nq * p.group <= p.small_rows) return;
    const float* part = p.partials + at * p.chunks * (D + 2);
    float m = kNothing;
    for (int c = 0; c < p.chunks; ++c) m = fmaxf(m, part[c * (D + 2) + D]);
    float l = 0.f, o[D / 32] = {};
    for (int c = 0; c < p.chunks; ++c) {
        const float f = ex2(part[c * (D + 2) + D] - m);
        l += f * part[c * (D + 2) + D + 1];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] += f * part[c * (D + 2) + lane + 32 * i];
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) store_out(p.out, at * D + lane + 32 * i, l == 0.f ? 0.f : o[i] / l, bf16 != 0);
}

}  // namespace
}  // namespace tq

#include "tq_attend8_stream.cuh"
#include "tq_attend8_prompt.cuh"

namespace tq {
namespace {

enum class Attend8Kind { kFew, kStream, kPrompt };

struct Attend8Plan {
    Attend8Kind kind;
    int nt, warps, chunks;              // warps of a CTA and CTAs of a cluster (kFew), parts of an item's keys (kPrompt)
    int64_t tiles;                      // of a sequence; of all sequences for kPrompt
    int small_rows;                     // kPrompt: sequences of at most so many rows are left to the persistent kernel
};

// The persistent kernel takes launches of so many pages, 14 for each warp of the GPU.  It gains by sharing out few long items, or a few more than fill
// the GPU once; where clusters fill it evenly they are ahead up to about 100000 pages, and one line by pages cannot have both.  In us, clusters / persistent,
// 64 / 8 heads, fp16, n sequences of so many tokens: above the line 64 x 1024 32.1 / 37.3, 64 x 2048 57.0 / 58.8, 64 x 4096 106.0 / 101.7, 1 x 65536
// 52.6 / 38.2, 16 x 4096 31.4 / 36.0, 20 x 4096 80.7 / 41.5; below it 64 x 512 19.2 / 25.5, 4 x 4096 13.7 / 18.4, 20 x 2048 43.5 / 27.8.
constexpr int64_t kStreamPages = 32768;

// Which kernel, and how it is cut.
Attend8Plan attend8_plan(int64_t num_rows, int64_t seqs, int kv_heads, int group, int max_queries, int max_pages) {
    Attend8Plan a = {};
    const int64_t rows = static_cast<int64_t>(group) * max_queries;
    // (64 x 8192 tokens, 64 / 8 heads: 32 rows are 428 to 440 us in tiles of 16 rows, 64 rows 667 in one tile of 256, both fp16.)
    if (rows > 32) {
        a.kind = Attend8Kind::kPrompt;
        a.tiles = (rows + 2 * kTile - 1) / (2 * kTile) * seqs;
        const int64_t full = num_rows * group / (2 * kTile);
        if (full + seqs < a.tiles) a.tiles = full + seqs;
        int64_t items = a.tiles;
        // Decodes next to a chunk: a tile of 256 rows with 4 or 8 in use costs what a full one does.  (32 / 8 heads, 64 decodes over 8192 tokens and a
        // chunk of 2048: 606 us, 1222 by one kernel; 200 over 1024 and two of 1024: 207, 639; 8 over 4096 and four of 512: 275, 288.)
        if (group <= 16 && num_rows < seqs * max_queries && seqs * kv_heads * max_pages >= kStreamPages) {
            a.small_rows = 16;
            a.nt = group <= 8 ? 1 : 2;
            items = full + 1;
        }
        items *= kv_heads;
        const int64_t steps = (max_pages + 2 * kTilePages - 1) / (2 * kTilePages);
        int64_t want = kMaxCtas / items;                                // parts per item, of two steps at least, that fill the GPU
        if (want > steps) want = steps;
        a.chunks = static_cast<int>(want < 1 ? 1 : want);
        return a;
    }
    a.nt = rows <= 8 ? 1 : 2;
    a.tiles = (rows + 8 * a.nt - 1) / (8 * a.nt);
    const int64_t items = seqs * kv_heads * a.tiles;
    a.kind = items * max_pages >= kStreamPages ? Attend8Kind::kStream : Attend8Kind::kFew;
    // One CTA of 16 warps (8 for 16 query rows) fits an SM, or four of 4.
    a.warps = items > kMaxCtas ? 4 : a.nt == 1 ? 16 : 8;
    a.chunks = 1;
    // Clusters lie within a part of the GPU: 35 of 4 CTAs and 16 of 8 fit next to one another, and a margin is left (16 of 8: 20.6 us, 16 of 4: 13).
    const int64_t fit[] = {0, 148, 74, 0, 32, 0, 0, 0, 12};
    while (a.chunks < kMaxCluster && items <= fit[a.chunks * 2] && a.chunks * a.warps < max_pages) a.chunks *= 2;
    return a;
}

int64_t attend8_workspace(const Attend8Plan& a, int64_t rows, int q_heads, int head_dim) {
    int64_t need = 0;
    if (a.kind == Attend8Kind::kStream || a.small_rows)
        need = 4 * (head_dim == 64 ? (a.nt == 1 ? StreamSpace<64, 1>::kFloats : StreamSpace<64, 2>::kFloats)
                                   : (a.nt == 1 ? StreamSpace<128, 1>::kFloats : StreamSpace<128, 2>::kFloats));
    if (a.kind == Attend8Kind::kPrompt && a.chunks > 1) {                 // after the persistent kernel, in the same place
        const int64_t parts = rows * q_heads * a.chunks * (head_dim + 2) * 4;
        if (parts > need) need = parts;
    }
    return need;
}

// The opt-in shared-memory size is a per-device function attribute; set once per device.
template <typename Kernel>
cudaError_t allow_shared_memory(Kernel kernel, int bytes, bool (&configured)[64]) {
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (configured[dev]) return cudaSuccess;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    configured[dev] = err == cudaSuccess;
    return err;
}

template <int D>
cudaError_t launch_merge(const Attend8Params& p, bool bf16, cudaStream_t stream) {
    return launch_chained(attend8_merge_kernel<D>, dim3(static_cast<unsigned>((static_cast<int64_t>(p.rows) * p.q_heads + 3) / 4)), dim3(128), 0, stream, p, static_cast<int>(bf16));
}

template <int D, int NT, bool BF16, int WARPS>
cudaError_t launch_few(const Attend8Params& p, cudaStream_t stream) {
    static bool configured[64] = {};
    auto kernel = attend8_few_kernel<D, NT, BF16, WARPS>;
    constexpr int kSmem = few_smem(D, NT, WARPS);
    const cudaError_t err = allow_shared_memory(kernel, kSmem, configured);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.chunks) * p.tiles * p.kv_heads * p.seqs));
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.chunks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.chunks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int D, int NT, bool BF16>
cudaError_t launch_stream(const Attend8Params& p, cudaStream_t stream) {
    static bool configured[64] = {};
    auto kernel = attend8_stream_kernel<D, NT, BF16>;
    cudaError_t err = allow_shared_memory(kernel, StreamSmem<D, NT>::kBytes, configured);
    if (err != cudaSuccess) return err;
    err = launch_chained(kernel, dim3(kMaxCtas), dim3(stream_warps(NT) * 32), StreamSmem<D, NT>::kBytes, stream, p);
    if (err != cudaSuccess) return err;
    return launch_chained(attend8_stream_merge_kernel<D, NT, BF16>, dim3(kMaxCtas - 1, NT), dim3(256), 0, stream, p);
}

template <int D, bool BF16>
cudaError_t launch_prompt(const Attend8Params& p, cudaStream_t stream) {
    static bool configured[64] = {};
    auto kernel = attend8_prompt_kernel<D, BF16>;
    cudaError_t err = allow_shared_memory(kernel, PromptSmem<D>::kBytes, configured);
    if (err != cudaSuccess) return err;
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.chunks) * p.tiles * p.kv_heads));
    err = launch_chained(kernel, grid, dim3(kPromptThreads), PromptSmem<D>::kBytes, stream, p);
    return err != cudaSuccess || p.chunks == 1 ? err : launch_merge<D>(p, BF16, stream);
}

template <int D, bool BF16>
cudaError_t launch_attend8(const Attend8Params& p, const Attend8Plan& a, cudaStream_t stream) {
    if (a.kind == Attend8Kind::kFew) {
        if (a.nt == 1) return a.warps == 4 ? launch_few<D, 1, BF16, 4>(p, stream) : launch_few<D, 1, BF16, 16>(p, stream);
        return a.warps == 4 ? launch_few<D, 2, BF16, 4>(p, stream) : launch_few<D, 2, BF16, 8>(p, stream);
    }
    if (a.kind == Attend8Kind::kStream || a.small_rows) {
        Attend8Params q = p;
        if (a.small_rows) q.zero_rest = 0;                              // the other kernel's
        const cudaError_t err = a.nt == 1 ? launch_stream<D, 1, BF16>(q, stream) : launch_stream<D, 2, BF16>(q, stream);
        if (err != cudaSuccess || a.kind == Attend8Kind::kStream) return err;
    }
    return launch_prompt<D, BF16>(p, stream);
}

}  // namespace
}  // namespace tq

extern "C" int64_t tq_attend8_workspace_bytes(int64_t num_rows, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int max_queries,
                                              int max_pages_per_seq) {
    using namespace tq;
    if (num_rows < 0 || num_seqs < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads || max_queries < 1 || max_pages_per_seq < 0)
        return TQ_ERR_ARG;
    if (head_dim != 64 && head_dim != 128) return TQ_ERR_UNSUPPORTED;
    if (num_seqs == 0) return 0;
    const Attend8Plan a = attend8_plan(num_rows, num_seqs, num_kv_heads, num_q_heads / num_kv_heads, max_queries, max_pages_per_seq);
    return attend8_workspace(a, num_rows, num_q_heads, head_dim);
}

extern "C" int tq_attend8_paged(void* out, const void* q, int io_dtype, const void* cache, int64_t num_blocks, int block_size,
                                const int32_t* block_tables, int64_t bt_stride, const int32_t* seq_lens, const int32_t* query_start_loc,
                                float sm_scale, void* workspace, int64_t workspace_bytes, int32_t* status, int64_t num_rows, int num_seqs,
                                int num_q_heads, int num_kv_heads, int head_dim, int max_queries, int max_pages_per_seq, int zero_rest,
                                tq_stream_t stream) {
    using namespace tq;
    if (num_rows < 0 || num_seqs < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads || num_blocks < 0 || max_queries < 1 ||
        max_pages_per_seq < 0 || bt_stride < 0)
        return TQ_ERR_ARG;
    if ((io_dtype != TQ_DTYPE_F16 && io_dtype != TQ_DTYPE_BF16) || (head_dim != 64 && head_dim != 128)) return TQ_ERR_UNSUPPORTED;
    if (block_size < kPageTokens || block_size % kPageTokens || num_blocks > INT32_MAX || num_rows > INT32_MAX) return TQ_ERR_UNSUPPORTED;
    if (max_pages_per_seq > (1 << 26) || static_cast<int64_t>(max_queries) * num_q_heads > (1 << 30)) return TQ_ERR_UNSUPPORTED;
    if (num_rows == 0) return TQ_OK;
    if (num_seqs == 0) {
        if (!zero_rest) return TQ_OK;
        if (!out) return TQ_ERR_ARG;
        return cudaMemsetAsync(out, 0, static_cast<size_t>(num_rows) * num_q_heads * head_dim * 2, stream) == cudaSuccess ? TQ_OK : TQ_ERR_LAUNCH;
    }
    if (!out || !q || !cache || !block_tables || !seq_lens || num_blocks == 0) return TQ_ERR_ARG;
    if (!query_start_loc && (num_rows < num_seqs || max_queries != 1)) return TQ_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache)) % 16) return TQ_ERR_ARG;
    const Attend8Plan a = attend8_plan(num_rows, num_seqs, num_kv_heads, num_q_heads / num_kv_heads, max_queries, max_pages_per_seq);
    double grid = static_cast<double>(a.tiles) * num_kv_heads * a.chunks * (a.kind == Attend8Kind::kPrompt ? 1 : num_seqs);
    if (a.kind == Attend8Kind::kPrompt && a.chunks > 1) grid = fmax(grid, static_cast<double>(num_rows) * num_q_heads / 4);
    if (grid > INT32_MAX - 1) return TQ_ERR_UNSUPPORTED;
    const int64_t need = attend8_workspace(a, num_rows, num_q_heads, head_dim);
    if (need && (!workspace || workspace_bytes < need)) return TQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return TQ_ERR_ARG;
    Attend8Params p = {};
    p.out = out; p.q = q; p.cache = static_cast<const uint8_t*>(cache); p.tables = block_tables; p.seq_lens = seq_lens; p.starts = query_start_loc;
    p.partials = static_cast<float*>(workspace); p.status = status; p.num_blocks = num_blocks; p.table_stride = bt_stride;
    p.scale_log2 = sm_scale * kLog2e; p.rows = static_cast<int>(num_rows); p.seqs = num_seqs; p.q_heads = num_q_heads; p.kv_heads = num_kv_heads;
    p.group = num_q_heads / num_kv_heads; p.pages_per_block = block_size / kPageTokens; p.max_pages = max_pages_per_seq; p.max_queries = max_queries;
    p.tiles = static_cast<int>(a.tiles); p.chunks = a.chunks; p.zero_rest = zero_rest; p.small_rows = a.small_rows;
    const bool bf16 = io_dtype == TQ_DTYPE_BF16;
    const cudaError_t err = head_dim == 64 ? (bf16 ? launch_attend8<64, true>(p, a, stream) : launch_attend8<64, false>(p, a, stream))
                                           : (bf16 ? launch_attend8<128, true>(p, a, stream) : launch_attend8<128, false>(p, a, stream));
    return err == cudaSuccess ? TQ_OK : TQ_ERR_LAUNCH;
}
