// Attention over the 8-bit cache for launches that fill the GPU with few query rows per sequence; included by tq_attend8.cu.
//
// One CTA of 16 warps (12 for 16 query rows) per SM.  The pages of all items - (sequence, KV head, tile of 8 NT query rows), in that order - are
// laid end to end and cut into one equal, contiguous share per warp, so that sequences of any lengths load all warps alike.  A warp
// copies its pages ahead with cp.async, 16 bytes a lane, into a ring of its own in shared memory: what is in flight is then
// bounded by shared memory (2 pages a warp, 128 KB an SM) and not by registers, which with one page of prefetch a warp reached
// 4.1 of 6.5 TB/s.  The 16-byte pieces of a row are placed under an XOR of their index so that both the reads of keys (8 lanes: two
// tokens, four pieces) and of values (four tokens two apart, two pieces) touch all banks once.
//
// 64 / 8 heads of 128, fp16, 64 sequences of 8192 tokens: 185 us = 5.8 TB/s, 0.89 of a copy; 64 uneven ones of bf16 74 us, 0.73.  What is missing: 4 us to the
// first page, CTAs that end within 6 % of one another, joins and merge (7 us).  359 warp instructions a page at half of the issue slots.
//
// Whole items are written from registers.  Parts are joined in shared memory by the CTA, and what crosses CTAs goes to the workspace, at
// most two parts a CTA, for a second kernel.
#pragma once

namespace tq {
namespace {

constexpr int kStages = 2;
constexpr int kGroups = 512;                    // entries of the prefix over sequences
__host__ __device__ constexpr int stream_warps(int nt) { return nt == 1 ? 16 : 12; }
constexpr int kMaxCtas = 148;

template <int D, int NT>
struct StreamSmem {
    static constexpr int kWarps = stream_warps(NT);
    static constexpr int kStage = 2 * kPageTokens * D;
    static constexpr int kRing = kStages * kStage;                       // of a warp; a part of 8 NT rows fits in it
    static constexpr int kPart = 8 * NT * D * 4;
    static constexpr int kFirst = kWarps * kRing;                        // first parts of warps that go on with another item
    static constexpr int kScales = kFirst + kWarps * kPart;              // [warps][stages] 16 bytes
    static constexpr int kPrefix = kScales + kWarps * kStages * 16;      // [groups + 1] int64
    static constexpr int kStats = kPrefix + (kGroups + 2) * 8;           // [warps][2][8 NT][2] floats: reference, denominator
    static constexpr int kEntries = kStats + kWarps * 2 * 8 * NT * 8;    // [warps][2] entries
    static constexpr int kBytes = kEntries + kWarps * 2 * 32;
    static_assert(kRing >= kPart, "a last part takes the place of the ring");
};

// A part of an item: its query rows, and whether it holds the item's first and last page.
struct alignas(16) PartEntry {
    int first_row, rows, r0, kvh;       // rows: of the sequence and KV head; r0: first one of the tile
    int valid, begins, ends, pad;
};

// Workspace: parts [ctas][2][8 NT][D], statistics [ctas][2][8 NT][2], entries [ctas][2].
template <int D, int NT>
struct StreamSpace {
    static constexpr int64_t kPart = 8 * NT * D;
    static constexpr int64_t kStats = kMaxCtas * 2 * kPart;
    static constexpr int64_t kEntries = kStats + kMaxCtas * 2 * 8 * NT * 2;
    static constexpr int64_t kFloats = kEntries + kMaxCtas * 2 * (sizeof(PartEntry) / 4);
};

struct SeqInfo {
    int first_row, nq, len, pages, tiles;
};

template <int NT>
__device__ __forceinline__ SeqInfo seq_info(const Attend8Params& p, int seq) {
    SeqInfo s;
    rows_of(p, seq, s.first_row, s.nq);
    if (p.small_rows && s.nq * p.group > p.small_rows) s.nq = 0;           // left to the kernel of prompt chunks
    s.len = p.seq_lens[seq];
    if (pages_of_length(s.len) > p.max_pages) s.len = p.max_pages * kPageTokens;
    s.tiles = (s.nq * p.group + 8 * NT - 1) / (8 * NT);
    s.pages = s.tiles ? pages_of_length(s.len) : 0;
    return s;
}

// A place in the sequence of all pages.
struct Cursor {
    int seq, kvh, tile, page;
    int pages, tiles;           // of the sequence
};

// The next item with pages.
template <int NT>
__device__ __forceinline__ void next_item(Cursor& c, const Attend8Params& p) {
    c.page = 0;
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.kvh < p.kv_heads) return;
    c.kvh = 0;
    c.pages = 0;
    while (c.pages == 0 && ++c.seq < p.seqs) {
        const SeqInfo s = seq_info<NT>(p, c.seq);
        c.pages = s.pages;
        c.tiles = s.tiles;
    }
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Byte of a row's 16-byte piece in a page's keys / values in shared memory.
template <int D>
__device__ __forceinline__ int key_byte(int row, int piece) {
    return D == 128 ? row * 128 + ((piece ^ ((row & 1) << 2)) << 4) : row * 64 + (piece << 4);
}
template <int D>
__device__ __forceinline__ int value_byte(int row, int piece) {
    if (D == 128) return row * 128 + ((piece ^ (((row >> 1) & 3) << 1)) << 4);
    return (row >> 1) * 128 + ((((row & 1) * 4 + piece) ^ (((row >> 1) & 3) << 1)) << 4);
}

// A lane copies one piece of rows r0, r0 + 4, ... of the keys, and of rows whose XOR is the same of the values, so that all
// addresses are a base of the lane and constants.
template <int D>
struct PageCopy {
    int key_from, key_to, value_from, value_to;
    __device__ __forceinline__ explicit PageCopy(int lane) {
        const int row = D == 128 ? lane >> 3 : lane >> 2, piece = D == 128 ? lane & 7 : lane & 3;
        key_from = row * D + piece * 16;
        key_to = key_byte<D>(row, piece);
        // D = 128: rows 2 r, 2 r + 1, 2 r + 8, 2 r + 9.  D = 64: rows r and r + 8.
        const int first = D == 128 ? 2 * row : row;
        value_from = (kPageTokens + first) * D + piece * 16;
        value_to = kPageTokens * D + value_byte<D>(first, piece);
    }
    __device__ __forceinline__ void operator()(uint32_t stage, uint32_t scales, const uint8_t* page, int lane) const {
#pragma unroll
        for (int i = 0; i < kPageTokens * D / 512; ++i) copy16(stage + key_to + i * 512, page + key_from + i * 512);
#pragma unroll
        for (int i = 0; i < kPageTokens * D / 512; ++i) {
            const int off = D == 128 ? (i & 1) * 128 + (i >> 1) * 1024 : i * 512;
            copy16(stage + value_to + off, page + value_from + off);
        }
        if (lane == 0) copy16(scales, page + cache8_scale_off(D));
    }
};

__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

template <int D>
__device__ __forceinline__ void read_keys(Page<D>& x, uint32_t stage, uint32_t scales, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) x.k[r][c] = lds16(stage + key_byte<D>(g + 8 * r, 4 * c + t));
    const uint2 s = lds8(scales);
    x.scales = make_float2(__uint_as_float(s.x), __uint_as_float(s.y));
}

template <int D>
__device__ __forceinline__ void read_values(Page<D>& x, uint32_t stage, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (D == 128) {
            const uint4 w = lds16(stage + kPageTokens * D + value_byte<D>(row, g));
            x.v[i][0] = w.x; x.v[i][1] = w.y; x.v[i][2] = w.z; x.v[i][3] = w.w;
        } else {
            const uint2 w = lds8(stage + kPageTokens * D + value_byte<D>(row, g >> 1) + 8 * (g & 1));
            x.v[i][0] = w.x; x.v[i][1] = w.y;
        }
    }
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(stream_warps(NT) * 32, 1) attend8_stream_kernel(const Attend8Params p) {
    using Smem = StreamSmem<D, NT>;
    using Space = StreamSpace<D, NT>;
    constexpr int W = stream_warps(NT), COLS = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    int64_t* prefix = reinterpret_cast<int64_t*>(smem + Smem::kPrefix);
    float* stats = reinterpret_cast<float*>(smem + Smem::kStats);
    PartEntry* entries = reinterpret_cast<PartEntry*>(smem + Smem::kEntries);
    __shared__ int64_t warp_sum[W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    if (tid < W * 2) entries[tid].valid = 0;
    pdl_wait();
    pdl_release();

    // Prefix of pages over groups of sequences, and what no page leads to: sequences without tokens, rows behind the last one, flags.
    const int per = (p.seqs + kGroups - 1) / kGroups;
    int64_t mine[(kGroups + W * 32 - 1) / (W * 32)];
    constexpr int kOwn = (kGroups + W * 32 - 1) / (W * 32);
    int64_t sum = 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        const int e = tid * kOwn + k;
        mine[k] = 0;
        for (int s = e * per; e < kGroups && s < min((e + 1) * per, p.seqs); ++s) {
            const SeqInfo i = seq_info<NT>(p, s);
            mine[k] += static_cast<int64_t>(i.pages) * i.tiles * p.kv_heads;
        }
        sum += mine[k];
    }
    {
        int64_t x = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        int64_t before = x - sum;
        for (int w = 0; w < warp; ++w) before += warp_sum[w];
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const int e = tid * kOwn + k;
            if (e < kGroups) prefix[e] = before;
            before += mine[k];
            if (e == kGroups - 1) prefix[kGroups] = before;
        }
    }
    __syncthreads();

    constexpr int kShares = kMaxCtas * W;
    const int64_t total = prefix[kGroups];
    const int share = blockIdx.x * W + warp;
    const int each = static_cast<int>(total / kShares), more = static_cast<int>(total - static_cast<int64_t>(each) * kShares);
    const int64_t from = static_cast<int64_t>(each) * share + min(more, share);
    const int count = each + (share < more);
    const uint32_t ring = smem_u32(smem) + warp * Smem::kRing, scales = smem_u32(smem) + Smem::kScales + warp * kStages * 16;
    if (count > 0) {
        Cursor c;
        {
            // Last group that begins at or before `from`, 32 and then 16 at a time.
            int lo = __popc(__ballot_sync(0xffffffffu, prefix[lane * (kGroups / 32)] <= from)) - 1;
            lo *= kGroups / 32;
            lo += __popc(__ballot_sync(0xffffffffu, lane < kGroups / 32 && prefix[lo + (lane & (kGroups / 32 - 1))] <= from)) - 1;
            int64_t rest = from - prefix[lo];
            for (c.seq = lo * per;; ++c.seq) {
                const SeqInfo s = seq_info<NT>(p, c.seq);
                const int64_t all = static_cast<int64_t>(s.pages) * s.tiles * p.kv_heads;
                if (rest < all) {
                    c.pages = s.pages;
                    c.tiles = s.tiles;
                    const int index = rest <= INT32_MAX ? static_cast<int>(rest) / s.pages : static_cast<int>(rest / s.pages);
                    c.page = static_cast<int>(rest - static_cast<int64_t>(index) * s.pages);
                    c.kvh = index / s.tiles;
                    c.tile = index - c.kvh * s.tiles;
                    break;
                }
                rest -= all;
            }
        }
        // The producer's side: a cursor of its own, and the blocks of 32 pages, one a lane.
        Cursor ahead = c;
        int to_copy = count, slot = 0, block = 0, in_window = 32, in_block = ahead.page % p.pages_per_block;
        bool bad = false;
        const PageCopy<D> copy(lane);
        const int64_t block_bytes = static_cast<int64_t>(p.kv_heads) * p.pages_per_block * cache8_page_bytes(D);
        const int head_bytes = p.pages_per_block * cache8_page_bytes(D);
        auto produce = [&]() {
            if (to_copy > 0) {
                if (in_window == 32) {
                    in_window = 0;
                    block = 0;
                    if (ahead.page + lane < ahead.pages) {
                        block = __ldg(p.tables + ahead.seq * p.table_stride + (ahead.page + lane) / p.pages_per_block);
                        if (block < 0 || block >= p.num_blocks) {
                            bad = true;
                            block = block < 0 ? 0 : static_cast<int>(p.num_blocks - 1);
                        }
                    }
                }
                const int b = __shfl_sync(0xffffffffu, block, in_window);
                copy(ring + slot * Smem::kStage, scales + slot * 16,
                     p.cache + b * block_bytes + static_cast<int64_t>(ahead.kvh) * head_bytes + in_block * cache8_page_bytes(D), lane);
                --to_copy;
                ++in_window;
                if (++in_block == p.pages_per_block) in_block = 0;
                if (++ahead.page == ahead.pages) {
                    next_item<NT>(ahead, p);
                    in_window = 32;
                    in_block = 0;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            slot = slot + 1 == kStages ? 0 : slot + 1;
        };
#pragma unroll
        for (int i = 0; i < kStages; ++i) produce();

        int stage = 0;
        int left = count;
        bool first = true;
        while (left > 0) {
            const SeqInfo s = seq_info<NT>(p, c.seq);
            const int kvh = c.kvh, r0 = c.tile * COLS, nrows = s.nq * p.group;
            const int a = c.page, b = min(s.pages - a, left) + a;
            Rows<D, NT> w;
            load_queries<D, NT, BF16>(w, p, s.first_row, kvh, r0, nrows, s.len, s.nq, lane);
            for (int page = a; page < b; ++page) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
                __syncwarp();
                Page<D> x;
                float sc[NT][4];
                uint32_t weights[NT][2];
                read_keys<D>(x, ring + stage * Smem::kStage, scales + stage * 16, lane);
                page_scores<D, NT>(sc, w, x);
                read_values<D>(x, ring + stage * Smem::kStage, lane);
                __syncwarp();
                produce();                                         // into the place just read
                page_weights<D, NT>(w, sc, x.scales, page, weights);
                page_products<D, NT>(w, x, weights, page, lane);
                stage = stage + 1 == kStages ? 0 : stage + 1;
            }
            left -= b - a;
            const bool whole = a == 0 && b == s.pages;
            float up[NT][2], l[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[n][j] = w.l[n][j];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], o);
                    up[n][j] = ex2(w.u[n][j] - w.m[n][j] - kHeadroom);
                }
            if (whole) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int row = r0 + 8 * n + 2 * t + j;
                        if (row >= nrows) continue;
                        const float f = l[n][j] == 0.f ? 0.f : up[n][j] / l[n][j];
                        const int token = row / p.group, head = kvh * p.group + row - token * p.group;
                        uint16_t* to = static_cast<uint16_t*>(p.out) + (static_cast<int64_t>(s.first_row + token) * p.q_heads + head) * D + D / 8 * g;
                        uint32_t v[D / 16];
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
                            v[i] = l[n][j] == 0.f ? 0u : pack_out(w.o[i][n][j] * f, w.o[i][n][j + 2] * f, BF16);
#pragma unroll
                        for (int i = 0; i < D / 16; i += 4) *reinterpret_cast<uint4*>(to + 2 * i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
            } else {
                // The last part of a warp takes the place of its ring, a first one behind which more comes has a place of its own.
                const int e = warp * 2 + (first ? 0 : 1);
                float* at = reinterpret_cast<float*>(smem + (first ? Smem::kFirst + warp * Smem::kPart : warp * Smem::kRing));
                __syncwarp();                                      // the ring has been read, and nothing is on its way to it
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int col = 8 * n + 2 * t + j;
#pragma unroll
                        for (int i = 0; i < D / 16; i += 2)
                            *reinterpret_cast<float4*>(at + col * D + D / 8 * g + 2 * i) =
                                make_float4(w.o[i][n][j] * up[n][j], w.o[i][n][j + 2] * up[n][j], w.o[i + 1][n][j] * up[n][j], w.o[i + 1][n][j + 2] * up[n][j]);
                        if (g == 0) {
                            stats[(e * COLS + col) * 2] = w.m[n][j];
                            stats[(e * COLS + col) * 2 + 1] = l[n][j];
                        }
                    }
                if (lane == 0) entries[e] = PartEntry{s.first_row, nrows, r0, kvh, 1, a == 0, b == s.pages, 0};
            }
            first = false;
            if (left > 0) next_item<NT>(c, p);
        }
        if (bad && p.status) atomicOr(p.status, TQ_STATUS_BAD_BLOCK);
    }
    __syncthreads();

    // Join the parts of items: lane e looks at entry e, an item's parts stand side by side (pages are contiguous), and a warp takes one query
    // row of one item at a time.
    const PartEntry mine_entry = entries[min(lane, 2 * W - 1)];
    const bool valid = lane < 2 * W && mine_entry.valid;
    const uint32_t there = __ballot_sync(0xffffffffu, valid), ending = __ballot_sync(0xffffffffu, valid && mine_entry.ends);
    const uint32_t before = there & ((1u << lane) - 1u);
    const uint32_t heads = __ballot_sync(0xffffffffu, valid && (before == 0 || (ending >> (31 - __clz(before)) & 1)));
    const int groups = __popc(heads);
    uint32_t left_heads = heads;
    int at_group = 0;
    for (int task = warp; task < groups * COLS; task += W) {
        const int group = task / COLS, col = task % COLS;
        for (; at_group < group; ++at_group) left_heads &= left_heads - 1;
        const int e0 = __ffs(left_heads) - 1;
        const uint32_t behind = left_heads & (left_heads - 1);
        const uint32_t members = there & ~((1u << e0) - 1u) & (behind ? (1u << (__ffs(behind) - 1)) - 1u : ~0u);
        const int e1 = 31 - __clz(members);
        const PartEntry head = entries[e0];
        const bool done = head.begins && (ending >> e1 & 1);
        const int row = head.r0 + col;
        if (row >= head.rows) continue;
        const bool member = members >> lane & 1;
        const float2 stat = member ? *reinterpret_cast<const float2*>(stats + (lane * COLS + col) * 2) : make_float2(kNothing, 0.f);
        float m = stat.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float f = ex2(stat.x - m);
        float l = member ? f * stat.y : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        // Parts four at a time; beyond the last one it is read again and left out.  A part whose weight is zero counts: a NaN in its values does.
        float o[D / 32] = {};
        const int offset = col * D + lane * (D / 32);
        for (uint32_t rest = members; rest;) {
            float part[4][D / 32], weight[4];
            bool more[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = rest ? __ffs(rest) - 1 : e1;
                weight[k] = __shfl_sync(0xffffffffu, f, e);
                more[k] = rest != 0;
                const float* at = reinterpret_cast<const float*>(smem + (e & 1 ? (e >> 1) * Smem::kRing : Smem::kFirst + (e >> 1) * Smem::kPart));
#pragma unroll
                for (int i = 0; i < D / 32; ++i) part[k][i] = at[offset + i];
                rest &= rest - 1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (more[k]) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) o[i] += weight[k] * part[k][i];
                }
        }
        if (done) {
            store_row<D, BF16>(p, head.first_row, head.kvh, row, o, l, lane);
        } else {
            const int64_t at = static_cast<int64_t>(blockIdx.x) * 2 + (head.begins ? 1 : 0);
            float* to = p.partials + at * Space::kPart + col * D + lane * (D / 32);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) to[i] = o[i];
            if (lane == 0) *reinterpret_cast<float2*>(p.partials + Space::kStats + (at * COLS + col) * 2) = make_float2(m, l);
        }
    }
    // What goes on in other CTAs: the first group where it does not begin here, the last one where it does not end here.
    if (warp == 0) {
        PartEntry* to = reinterpret_cast<PartEntry*>(p.partials + Space::kEntries) + blockIdx.x * 2;
        const int first = there ? __ffs(there) - 1 : 0, last = there ? 31 - __clz(there) : 0, last_head = heads ? 31 - __clz(heads) : 0;
        if (lane < 2) {
            // side 0: goes on from the CTA before; side 1: begins here and goes on
            PartEntry e = entries[lane == 0 ? first : last_head];
            const bool ends = lane == 0 ? groups > 1 || entries[last].ends : entries[last].ends;
            e.ends = ends;
            e.valid = there && (lane == 0 ? !e.begins : e.begins && !ends);
            to[lane] = e;
        }
    }

    const int row_words = p.q_heads * D / 2;
    if (p.zero_rest && blockIdx.x == 0) zero_ends<D>(p);
    for (int s = blockIdx.x; s < p.seqs; s += gridDim.x) {
        const SeqInfo i = seq_info<NT>(p, s);
        if (!i.pages) zero_rows<D>(p, i.first_row, i.first_row + i.nq);
        int first_row, nq;
        const int left_out = rows_of(p, s, first_row, nq);
        if (left_out && p.zero_rest) zero_rows<D>(p, first_row + nq, first_row + nq + left_out);
        if (tid == 0 && p.status) {
            const bool too_long = pages_of_length(p.seq_lens[s]) > p.max_pages;
            if (left_out || too_long) atomicOr(p.status, (too_long ? TQ_STATUS_BAD_BLOCK : 0) | (left_out ? TQ_STATUS_TOO_LONG : 0));
        }
    }
}

// Items that cross CTAs: block x takes the one that begins in CTA x and goes on, a warp per query row.  The entries and statistics of 32
// CTAs, and the parts of the first four, are asked for before it is known which of them matter.
template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(256) attend8_stream_merge_kernel(const Attend8Params p) {
    using Space = StreamSpace<D, NT>;
    constexpr int COLS = 8 * NT;
    pdl_release();
    pdl_wait();
    const int lane = threadIdx.x & 31, cta = blockIdx.x, col = blockIdx.y * 8 + (threadIdx.x >> 5);
    const PartEntry* entries = reinterpret_cast<const PartEntry*>(p.partials + Space::kEntries);
    const float2* stats = reinterpret_cast<const float2*>(p.partials + Space::kStats);
    const PartEntry head = entries[cta * 2 + 1];
    float m = kNothing, l = 0.f, o[D / 32] = {};
    constexpr int kEarly = 4;
    float early[kEarly][D / 32];
#pragma unroll
    for (int i = 0; i < kEarly; ++i) {
        const float* from = p.partials + (min(cta + i, kMaxCtas - 1) * 2 + (i == 0)) * Space::kPart + col * D + lane * (D / 32);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) early[i][d] = from[d];
    }
    bool over = false;
    for (int base = cta; base < kMaxCtas && !over; base += 32) {
        const int c = base + lane, side = c == cta ? 1 : 0;
        // side 0 of a following CTA belongs to this item up to the one that holds its end
        const bool in = c < kMaxCtas;
        const int ends = in && c > cta ? entries[c * 2].ends : !in;
        const float2 mine = in ? stats[(c * 2 + side) * COLS + col] : make_float2(kNothing, 0.f);
        if (base == cta && (!head.valid || head.r0 + col >= head.rows)) return;
        const uint32_t hit = __ballot_sync(0xffffffffu, ends);
        const int n = hit ? __ffs(hit) - (__shfl_sync(0xffffffffu, in, __ffs(hit) - 1) ? 0 : 1) : 32;
        over = hit != 0;
        const float2 stat = lane < n ? mine : make_float2(kNothing, 0.f);
        float most = fmaxf(stat.x, m);
#pragma unroll
        for (int k = 16; k; k >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k));
        const float down = ex2(m - most), f = ex2(stat.x - most);
        l = l * down + (lane < n ? f * stat.y : 0.f);                 // this lane's share
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= down;
        m = most;
        int k = 0;
        if (base == cta) {
#pragma unroll
            for (int i = 0; i < kEarly; ++i) {
                if (i < n) {
                    const float fk = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
                    for (int d = 0; d < D / 32; ++d) o[d] += fk * early[i][d];
                }
            }
            k = kEarly;
        }
#pragma unroll 8
        for (; k < n; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const float* from = p.partials + ((base + k) * 2 + (base + k == cta)) * Space::kPart + col * D + lane * (D / 32);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] += fk * from[i];
        }
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
    store_row<D, BF16>(p, head.first_row, head.kvh, head.r0 + col, o, l, lane);
}

}  // namespace
}  // namespace tq
