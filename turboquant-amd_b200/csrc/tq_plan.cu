// Step tables of a paged cache, built on the GPU from the requests' lengths.
//
// plan: request i holds context_i tokens and brings query_i new ones.  It needs ceil((context + query) / B) - ceil(context / B) further
// blocks of B tokens, which come from the top of a stack of free ones in the order of the requests.  Out of it come the extended
// block tables, the slot and the position of every new token, the new lengths, the rows' offsets and the new height of the stack.
// release: the blocks of ended requests go back on the stack, in order.
//
// Both are a prefix sum over the requests with an expansion behind it.  Every CTA does the whole sum by itself, 2048 requests at
// a time (16 KB from L2), and then expands its own share of the rows: no CTA waits for another one, there is one launch, and the
// order in which blocks are given out does not depend on timing.  Bound: latency (launch, lengths, scan, search, store): 64 requests
// 5.1 us and 1000 with 107000 rows 6.8 to plan, 3.5 and 4.9 to release (in a graph).
#include "tq_common.cuh"

namespace tq {
namespace {

constexpr int kThreads = 512;
constexpr int kPer = 4;                          // consecutive requests of a thread
constexpr int kChunk = kThreads * kPer;

// Exclusive sums over the block of two values per thread; the totals come back in `total`.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t (&total)[2], int64_t (*warp_sums)[kThreads / 32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = a, y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) {
            x += u;
            y += v;
        }
    }
    __syncthreads();                             // the sums of the chunk before have been read
    if (lane == 31) {
        warp_sums[0][warp] = x;
        warp_sums[1][warp] = y;
    }
    __syncthreads();
    int64_t before[2] = {0, 0};
    total[0] = total[1] = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        const int64_t u = warp_sums[0][w], v = warp_sums[1][w];
        if (w < warp) {
            before[0] += u;
            before[1] += v;
        }
        total[0] += u;
        total[1] += v;
    }
    a = before[0] + x - a;
    b = before[1] + y - b;
}

// Blocks of n tokens: lengths fit 31 bits, and a 64-bit division takes a hundred instructions.
__device__ __forceinline__ int blocks_of(int n, int block_size) {
    return static_cast<int>((static_cast<uint32_t>(n) + static_cast<uint32_t>(block_size) - 1u) / static_cast<uint32_t>(block_size));
}

struct PlanParams {
    const int32_t* query_lens;
    const int32_t* context_lens;
    int32_t* tables;
    const int32_t* free_blocks;
    const int32_t* free_count;
    int64_t* slots;
    int64_t* positions;
    int32_t* seq_lens;
    int32_t* starts;
    int32_t* new_count;
    int32_t* status;
    int64_t table_stride;
    int requests, width, block_size, rows, free_size;
};

__global__ void __launch_bounds__(kThreads) plan_kernel(const PlanParams p) {
    __shared__ int64_t sums[2][kThreads / 32];
    __shared__ int row_end[kChunk];              // rows of all requests up to and with this one, at most 2^31 - 1
    __shared__ int first_free[kChunk];           // place on the stack of the request's first new block; -1: it is not served
    __shared__ int context[kChunk];
    pdl_wait();
    pdl_release_if_small();
    const int count = min(max(*p.free_count, 0), p.free_size);
    const int per_cta = (p.rows + gridDim.x - 1) / gridDim.x;
    const int row_a = min(static_cast<int64_t>(blockIdx.x) * per_cta, static_cast<int64_t>(p.rows));
    const int row_b = min(static_cast<int64_t>(row_a) + per_cta, static_cast<int64_t>(p.rows));
    const bool writes = blockIdx.x == 0;
    int64_t rows_before = 0, blocks_before = 0;
    int64_t taken = 0;
    int flags = 0;

    for (int c0 = 0; c0 < p.requests; c0 += kChunk) {
        int64_t ctx[kPer], query[kPer], need[kPer], sum_rows = 0, sum_need = 0;
        bool wide[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = c0 + threadIdx.x * kPer + j;
            ctx[j] = i < p.requests ? max(p.context_lens[i], 0) : 0;
            query[j] = i < p.requests ? max(p.query_lens[i], 0) : 0;
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int64_t tokens = ctx[j] + query[j];
            const int total = tokens <= INT32_MAX ? blocks_of(static_cast<int>(tokens), p.block_size) : 0;
            wide[j] = tokens <= INT32_MAX && total <= p.width;
            need[j] = wide[j] ? total - blocks_of(static_cast<int>(ctx[j]), p.block_size) : 0;
            sum_rows += query[j];
            sum_need += need[j];
        }
        int64_t totals[2], at_row = sum_rows, at_block = sum_need;
        block_scan2(at_row, at_block, totals, sums);
        at_row += rows_before;
        at_block += blocks_before;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int slot = threadIdx.x * kPer + j, i = c0 + slot;
            at_row += query[j];
            const int64_t first = at_block;
            at_block += need[j];
            // What does not fit the rows is followed by nothing that fits them and needs a block, so that counting its blocks changes nothing.
            const bool fits = wide[j] && at_row <= p.rows;
            const bool served = fits && (need[j] == 0 || at_block <= count);
            if (served && need[j] > 0) taken = max(taken, at_block);
            if (i < p.requests && query[j] > 0) flags |= !fits ? TQ_STATUS_TOO_LONG : !served ? TQ_STATUS_NO_BLOCKS : 0;
            const int end = static_cast<int>(min(at_row, static_cast<int64_t>(p.rows)));
            row_end[slot] = i < p.requests ? end : INT32_MAX;
            first_free[slot] = served ? count - 1 - static_cast<int>(min(first, static_cast<int64_t>(count))) + 1 : -1;   // one above: 0 .. count
            context[slot] = static_cast<int>(ctx[j]);
            if (writes && i < p.requests) {
                p.starts[i + 1] = end;
                p.seq_lens[i] = static_cast<int>(served ? ctx[j] + query[j] : ctx[j]);
            }
        }
        __syncthreads();
        const int chunk_a = static_cast<int>(min(rows_before, static_cast<int64_t>(p.rows)));
        rows_before += totals[0];
        blocks_before += totals[1];
        const int chunk_b = static_cast<int>(min(rows_before, static_cast<int64_t>(p.rows)));
        for (int r = max(row_a, chunk_a) + threadIdx.x; r < min(row_b, chunk_b); r += kThreads) {
            int lo = 0, hi = min(kChunk, p.requests - c0) - 1;                 // first request whose rows end after r
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (row_end[mid] > r) hi = mid;
                else lo = mid + 1;
            }
            const int begin = lo ? row_end[lo - 1] : chunk_a;
            const int64_t pos = static_cast<int64_t>(context[lo]) + (r - begin);
            int64_t slot = -1;
            if (first_free[lo] >= 0) {
                // a request that is served ends before 2^31
                const int at = static_cast<int>(static_cast<uint32_t>(pos) / static_cast<uint32_t>(p.block_size)), in_block = static_cast<int>(pos) - at * p.block_size;
                const int held = blocks_of(context[lo], p.block_size);
                int32_t* entry = p.tables + (c0 + lo) * p.table_stride + at;
                int32_t block;
                if (at >= held) {
                    block = p.free_blocks[first_free[lo] - 1 - (at - held)];
                    if (in_block == 0) *entry = block;                         // every new block begins with a new token
                } else {
                    block = *entry;
                }
                if (block >= 0) slot = static_cast<int64_t>(block) * p.block_size + in_block;
            }
            p.slots[r] = slot;
            p.positions[r] = pos;
        }
        __syncthreads();
    }
    const int used = static_cast<int>(min(rows_before, static_cast<int64_t>(p.rows)));
    for (int r = max(row_a, used) + threadIdx.x; r < row_b; r += kThreads) {   // rows behind the last request
        p.slots[r] = -1;
        p.positions[r] = 0;
    }
    if (writes) {
        flags = __reduce_or_sync(0xffffffffu, flags);
        if ((threadIdx.x & 31) == 0 && flags && p.status) atomicOr(p.status, flags);
        // taken is at most count: a maximum over the block by way of the warps' sums
        const int most = __reduce_max_sync(0xffffffffu, static_cast<int>(taken));
        if ((threadIdx.x & 31) == 0) sums[0][threadIdx.x >> 5] = most;
        __syncthreads();
        if (threadIdx.x == 0) {
            int64_t all = 0;
            for (int w = 0; w < kThreads / 32; ++w) all = max(all, sums[0][w]);
            *p.new_count = count - static_cast<int>(all);
            p.starts[0] = 0;
        }
    }
}

struct ReleaseParams {
    const uint8_t* ended;
    const int32_t* context_lens;
    const int32_t* tables;
    int32_t* free_blocks;
    const int32_t* free_count;
    int32_t* lens;
    int32_t* new_count;
    int32_t* status;
    int64_t table_stride;
    int requests, width, block_size, free_size;
};

__global__ void __launch_bounds__(kThreads) release_kernel(const ReleaseParams p) {
    __shared__ int64_t sums[2][kThreads / 32];
    __shared__ int64_t place[kChunk];            // of the request's first block on the stack
    __shared__ int held[kChunk];
    pdl_wait();
    pdl_release_if_small();
    const int count = min(max(*p.free_count, 0), p.free_size);
    const bool writes = blockIdx.x == 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t before = 0;
    int flags = 0;
    for (int c0 = 0; c0 < p.requests; c0 += kChunk) {
        int64_t give[kPer], sum = 0, zero = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = c0 + threadIdx.x * kPer + j;
            const bool ends = i < p.requests && p.ended[i];
            const int64_t ctx = i < p.requests ? p.context_lens[i] : 0;
            give[j] = ends && ctx > 0 ? blocks_of(static_cast<int>(ctx), p.block_size) : 0;
            if (give[j] > p.width) {
                give[j] = p.width;
                flags |= TQ_STATUS_TOO_LONG;
            }
            sum += give[j];
            if (writes && i < p.requests) p.lens[i] = ends ? 0 : static_cast<int>(ctx);
        }
        int64_t totals[2], at = sum;
        block_scan2(at, zero, totals, sums);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            place[threadIdx.x * kPer + j] = count + before + at;
            held[threadIdx.x * kPer + j] = static_cast<int>(give[j]);
            at += give[j];
        }
        before += totals[0];
        __syncthreads();
        const int n = min(kChunk, p.requests - c0);
        for (int i = blockIdx.x * (kThreads / 32) + warp; i < n; i += gridDim.x * (kThreads / 32)) {
            const int32_t* from = p.tables + (c0 + i) * p.table_stride;
            const int64_t to = place[i];
            const int n = static_cast<int>(min(static_cast<int64_t>(held[i]), p.free_size - to));
#pragma unroll 4
            for (int j = lane; j < n; j += 32) p.free_blocks[to + j] = __ldg(from + j);
        }
        __syncthreads();
    }
    if (writes) {
        if (count + before > p.free_size) flags |= TQ_STATUS_TOO_LONG;
        flags = __reduce_or_sync(0xffffffffu, flags);
        if (lane == 0 && flags && p.status) atomicOr(p.status, flags);
        if (threadIdx.x == 0) *p.new_count = static_cast<int>(min(count + before, static_cast<int64_t>(p.free_size)));
    }
}

}  // namespace
}  // namespace tq

extern "C" int tq_plan_step(const int32_t* query_lens, const int32_t* context_lens, int32_t* block_tables, int64_t bt_stride,
                            const int32_t* free_blocks, const int32_t* free_count, int64_t* slot_mapping, int64_t* positions, int32_t* seq_lens,
                            int32_t* query_start_loc, int32_t* new_free_count, int32_t* status, int64_t num_requests, int64_t table_width,
                            int64_t num_free, int block_size, int64_t num_rows, tq_stream_t stream) {
    using namespace tq;
    if (num_requests < 0 || num_rows < 0 || num_free < 0 || table_width < 0 || bt_stride < 0 || block_size < 1) return TQ_ERR_ARG;
    if (num_requests > (1 << 24) || num_rows > (1 << 30) || num_free > INT32_MAX || table_width > INT32_MAX) return TQ_ERR_UNSUPPORTED;
    if (!free_count || !query_start_loc || !new_free_count) return TQ_ERR_ARG;
    if (num_requests && (!query_lens || !context_lens || !seq_lens || (table_width && !block_tables))) return TQ_ERR_ARG;
    if ((num_rows && (!slot_mapping || !positions)) || (num_free && !free_blocks)) return TQ_ERR_ARG;
    PlanParams p = {};
    p.query_lens = query_lens; p.context_lens = context_lens; p.tables = block_tables; p.free_blocks = free_blocks; p.free_count = free_count;
    p.slots = slot_mapping; p.positions = positions; p.seq_lens = seq_lens; p.starts = query_start_loc; p.new_count = new_free_count;
    p.status = status; p.table_stride = bt_stride; p.requests = static_cast<int>(num_requests); p.width = static_cast<int>(table_width);
    p.block_size = block_size; p.rows = static_cast<int>(num_rows); p.free_size = static_cast<int>(num_free);
    const int64_t share = (num_rows + kThreads - 1) / kThreads;
    const unsigned grid = static_cast<unsigned>(share < 1 ? 1 : share > 148 ? 148 : share);
    const cudaError_t err = launch_chained(plan_kernel, dim3(grid), dim3(kThreads), 0, stream, p);
    return err == cudaSuccess ? TQ_OK : TQ_ERR_LAUNCH;
}

extern "C" int tq_release_blocks(const uint8_t* ended, const int32_t* context_lens, const int32_t* block_tables, int64_t bt_stride,
                                 int32_t* free_blocks, const int32_t* free_count, int32_t* new_context_lens, int32_t* new_free_count, int32_t* status,
                                 int64_t num_requests, int64_t table_width, int64_t num_free, int block_size, tq_stream_t stream) {
    using namespace tq;
    if (num_requests < 0 || num_free < 0 || table_width < 0 || bt_stride < 0 || block_size < 1) return TQ_ERR_ARG;
    if (num_requests > (1 << 24) || num_free > INT32_MAX || table_width > INT32_MAX) return TQ_ERR_UNSUPPORTED;
    if (!free_count || !new_free_count || (num_free && !free_blocks)) return TQ_ERR_ARG;
    if (num_requests && (!ended || !context_lens || !new_context_lens || (table_width && !block_tables))) return TQ_ERR_ARG;
    ReleaseParams p = {};
    p.ended = ended; p.context_lens = context_lens; p.tables = block_tables; p.free_blocks = free_blocks; p.free_count = free_count;
    p.lens = new_context_lens; p.new_count = new_free_count; p.status = status; p.table_stride = bt_stride;
    p.requests = static_cast<int>(num_requests); p.width = static_cast<int>(table_width); p.block_size = block_size;
    p.free_size = static_cast<int>(num_free);
    const int64_t warps = kThreads / 32, share = (num_requests + warps - 1) / warps;
    const unsigned grid = static_cast<unsigned>(share < 1 ? 1 : share > 148 ? 148 : share);
    const cudaError_t err = launch_chained(release_kernel, dim3(grid), dim3(kThreads), 0, stream, p);
    return err == cudaSuccess ? TQ_OK : TQ_ERR_LAUNCH;
}
