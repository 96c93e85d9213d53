// New K/V rows into the 8-bit paged cache: e4m3 codes with one power-of-two scale per page of 16 tokens, head and K / V.
//
//   scale = 2^e, e the smallest with |x| <= 448 * 2^e over the finite values x of the page's rows, code = e4m3(x / scale)
//
// A page that a call begins (its first slot is among the call's rows) takes its scale from these rows.  One that is continued keeps
// the larger of its old scale and that of the new rows, and when it grows, the codes already there are rescaled.  The scale is a power of two so
// that this is exact but for codes that become subnormal: the relative precision of e4m3 does not depend on the scale.
//
// A run is a stretch of consecutive rows whose slots follow one another inside a page; one warp owns a run of one head's K or V:
// it holds the rows in registers between the maximum and the conversion, so each value is read once and written once.  Bound: HBM for
// prompts; for the few rows of a decode step the chain slot -> old scale and row -> maximum -> store.
// 8 heads of 128, bf16: 24 prompts, 55600 rows, 68.5 us = 0.76 of a copy with the 16 warps an SM that their registers allow (with fewer
// registers 24 warps took 79 us and 32 took 87); 64 single rows 2.4 us, 2000 single rows 11.9 (23 with one row in flight).
#include "tq_cache8.cuh"

namespace tq {
namespace {

struct Quantize8Params {
    const void* key;
    const void* value;
    uint8_t* cache;
    const int64_t* slots;
    int32_t* status;
    int64_t k_token, k_head, v_token, v_head;   // strides in elements
    int64_t n_slots;
    int n_tokens, heads, pages_per_block, window;
};

constexpr int kWarps = 8;

// Eight values of a row as fp32, from 16 bytes (fp16, bf16) or 32 (fp32).
template <int DTYPE>
struct Raw {
    uint4 v[DTYPE == TQ_DTYPE_F32 ? 2 : 1];
};
template <int DTYPE>
__device__ __forceinline__ void to_floats(const Raw<DTYPE>& r, float (&x)[8]) {
    if constexpr (DTYPE == TQ_DTYPE_F32) {
        const uint32_t w[8] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w, r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
        const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DTYPE == TQ_DTYPE_F16) {
                const float2 f = unpack_half2(w[i]);
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

// Largest finite value of a lane's eights as bits.  fmaxf passes a NaN over; an infinity is left out, which nothing but a second look can do.
template <int DTYPE, int N>
__device__ __forceinline__ uint32_t largest_finite(const Raw<DTYPE> (&raw)[N]) {
    const float infinity = __uint_as_float(0x7f800000u);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float x[8];
        to_floats<DTYPE>(raw[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
    }
    if (__any_sync(0xffffffffu, amax == infinity)) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float x[8];
            to_floats<DTYPE>(raw[i], x);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]) == infinity ? 0.f : fabsf(x[j]));
        }
    }
    return __float_as_uint(amax);
}

template <int DTYPE>
__device__ __forceinline__ void store_codes(uint8_t* to, const Raw<DTYPE>& raw, float inv) {
    float x[8];
    to_floats<DTYPE>(raw, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= inv;
    *reinterpret_cast<uint2*>(to) = make_uint2(e4m3x2(x[0], x[1]) | e4m3x2(x[2], x[3]) << 16, e4m3x2(x[4], x[5]) | e4m3x2(x[6], x[7]) << 16);
}

// Eight codes times a power of two, in place.
__device__ __forceinline__ void rescale_codes(uint8_t* at, float shrink) {
    const uint2 c = *reinterpret_cast<const uint2*>(at);
    const uint32_t w[2] = {c.x, c.y};
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float2 a = unpack_half2(e4m3x2_to_half2(w[j] & 0xffffu)), b = unpack_half2(e4m3x2_to_half2(w[j] >> 16));
        o[j] = e4m3x2(a.x * shrink, a.y * shrink) | e4m3x2(b.x * shrink, b.y * shrink) << 16;
    }
    *reinterpret_cast<uint2*>(at) = make_uint2(o[0], o[1]);
}

template <int D, int DTYPE>
__device__ __forceinline__ uint8_t* page_of_slot(const Quantize8Params& p, int64_t slot, int head) {
    const int64_t page = slot / kPageTokens;
    int64_t block;                                  // a 64-bit division takes a hundred instructions
    if (page <= 0x7fffffff) block = static_cast<uint32_t>(page) / static_cast<uint32_t>(p.pages_per_block);
    else block = page / p.pages_per_block;
    return p.cache + ((block * p.heads + head) * p.pages_per_block + (page - block * p.pages_per_block)) * static_cast<int64_t>(cache8_page_bytes(D));
}

template <int D, int DTYPE>
__global__ void __launch_bounds__(kWarps * 32) quantize8_kernel(const Quantize8Params p) {
    pdl_wait();
    pdl_release_if_small();
    constexpr int kLanes = D / 8;                   // lanes of a row
    constexpr int kRows = 32 / kLanes;              // rows at a time
    constexpr int kSteps = kPageTokens / kRows;
    constexpr int kItem = DTYPE == TQ_DTYPE_F32 ? 4 : 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / kLanes, col = lane % kLanes;
    const int per_run = 2 * p.heads;
    // Lane l looks at row r0 - 1 + l: runs that begin in the window end 16 rows after it at the latest.
    auto ask_slot = [&](int64_t window) {
        const int64_t mine = window * p.window - 1 + lane;
        return mine >= 0 && mine < p.n_tokens ? __ldg(p.slots + mine) : -1ll;
    };
    int64_t next_slot = ask_slot(blockIdx.x);
    for (int64_t window = blockIdx.x; window * p.window < p.n_tokens; window += gridDim.x) {
        const int64_t r0 = window * p.window, slot = next_slot;
        next_slot = ask_slot(window + gridDim.x);
        const bool valid = slot >= 0 && slot < p.n_slots;
        const int64_t before = __shfl_up_sync(0xffffffffu, slot, 1);
        const bool joins = valid && lane > 0 && slot == before + 1 && slot % kPageTokens != 0;
        const uint32_t joined = __ballot_sync(0xffffffffu, joins);
        const uint32_t in_window = ((1u << p.window) - 1u) << 1;
        const uint32_t starts = __ballot_sync(0xffffffffu, valid && !joins) & in_window;
        const uint32_t beyond = __ballot_sync(0xffffffffu, slot >= p.n_slots) & in_window;
        if (beyond && p.status && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(p.status, TQ_STATUS_BAD_SLOT);
        const int tasks = __popc(starts) * per_run;

        if (!(joined & starts << 1)) {
            // Runs of one row, as a decode step has them: a row for each D / 8 lanes, four in flight.
            constexpr int kFlight = 4;
            const int groups = kWarps * kRows * gridDim.y;
            for (int task0 = (blockIdx.y * kWarps + warp) * kRows; task0 < tasks; task0 += kFlight * groups) {      // the same for the whole warp
                Raw<DTYPE> raw[kFlight][1];
                uint8_t* codes[kFlight];
                uint32_t* scale[kFlight];
                uint32_t old[kFlight];
                int off[kFlight];
#pragma unroll
                for (int k = 0; k < kFlight; ++k) {
                    const int task = task0 + k * groups + sub;
                    const bool there = task < tasks;
                    const int run = there ? task / per_run : 0, rest = there ? task - run * per_run : 0, is_v = rest & 1, head = rest >> 1;
                    uint32_t left = starts;
                    for (int i = 0; i < run; ++i) left &= left - 1;
                    const int at = left ? __ffs(left) - 1 : 0;
                    const int64_t first = __shfl_sync(0xffffffffu, slot, at);
                    codes[k] = nullptr;
                    raw[k][0].v[0] = make_uint4(0, 0, 0, 0);
                    if constexpr (DTYPE == TQ_DTYPE_F32) raw[k][0].v[1] = make_uint4(0, 0, 0, 0);
                    if (there) {
                        uint8_t* base = page_of_slot<D, DTYPE>(p, first, head);
                        off[k] = static_cast<int>(first % kPageTokens);
                        codes[k] = base + is_v * kPageTokens * D + col * 8;
                        scale[k] = reinterpret_cast<uint32_t*>(base + cache8_scale_off(D)) + is_v;
                        const uint4* src = reinterpret_cast<const uint4*>(
                            static_cast<const uint8_t*>(is_v ? p.value : p.key) +
                            ((r0 - 1 + at) * (is_v ? p.v_token : p.k_token) + head * (is_v ? p.v_head : p.k_head) + col * 8) * kItem);
                        raw[k][0].v[0] = __ldg(src);
                        if constexpr (DTYPE == TQ_DTYPE_F32) raw[k][0].v[1] = __ldg(src + 1);
                        old[k] = *scale[k];
                    }
                }
#pragma unroll
                for (int k = 0; k < kFlight; ++k) {
                    uint32_t bits = largest_finite<DTYPE, 1>(raw[k]);
#pragma unroll
                    for (int o = kLanes / 2; o; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
                    if (!codes[k]) continue;
                    const int was = off[k] ? exponent_of_scale_bits(old[k]) : kMinExponent, e = max(was, scale_exponent_of_bits(bits));
                    if (e > was && off[k]) {
                        const float shrink = exp2_int(max(was - e, -126));
                        for (int r = 0; r < off[k]; ++r) rescale_codes(codes[k] + r * D, shrink);
                    }
                    store_codes<DTYPE>(codes[k] + off[k] * D, raw[k][0], exp2_int(-e));
                    if (col == 0) *scale[k] = static_cast<uint32_t>(127 + e) << 23;
                }
            }
            continue;
        }

        for (int task = blockIdx.y * kWarps + warp; task < tasks; task += kWarps * gridDim.y) {
            const int run = task / per_run, rest = task - run * per_run, is_v = rest & 1, head = rest >> 1;
            uint32_t left = starts;
            for (int i = 0; i < run; ++i) left &= left - 1;
            const int at = __ffs(left) - 1;                                        // the run's first lane
            const int64_t first = __shfl_sync(0xffffffffu, slot, at);
            const int len = __ffs(~(at == 31 ? 0u : joined >> (at + 1)));         // 1 .. 16: a page's first slot joins nothing
            const int off = static_cast<int>(first % kPageTokens);
            uint8_t* base = page_of_slot<D, DTYPE>(p, first, head);
            uint8_t* codes = base + is_v * kPageTokens * D + col * 8;
            uint32_t* scale = reinterpret_cast<uint32_t*>(base + cache8_scale_off(D)) + is_v;

            const uint8_t* rows = static_cast<const uint8_t*>(is_v ? p.value : p.key);
            const int64_t token = (is_v ? p.v_token : p.k_token) * kItem;
            rows += ((r0 - 1 + at + sub) * token) + (head * (is_v ? p.v_head : p.k_head) + col * 8) * kItem;
            Raw<DTYPE> raw[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (i * kRows + sub < len) {
                    const uint4* src = reinterpret_cast<const uint4*>(rows + i * kRows * token);
                    raw[i].v[0] = __ldg(src);
                    if constexpr (DTYPE == TQ_DTYPE_F32) raw[i].v[1] = __ldg(src + 1);
                } else {
                    raw[i].v[0] = make_uint4(0, 0, 0, 0);
                    if constexpr (DTYPE == TQ_DTYPE_F32) raw[i].v[1] = make_uint4(0, 0, 0, 0);
                }
            }
            const int old = off ? exponent_of_scale_bits(*scale) : kMinExponent;
            const uint32_t bits = __reduce_max_sync(0xffffffffu, largest_finite<DTYPE, kSteps>(raw));
            const int e = max(old, scale_exponent_of_bits(bits));
            const float inv = exp2_int(-e);
            if (e > old && off) {
                const float shrink = exp2_int(max(old - e, -126));
                for (int r = sub; r < off; r += kRows) rescale_codes(codes + r * D, shrink);
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (i * kRows + sub < len) store_codes<DTYPE>(codes + (off + i * kRows + sub) * D, raw[i], inv);
            if (lane == 0) *scale = static_cast<uint32_t>(127 + e) << 23;
        }
    }
}

template <int D>
cudaError_t launch_quantize8(const Quantize8Params& p, int dtype, dim3 grid, cudaStream_t stream) {
    const dim3 block(kWarps * 32);
    if (dtype == TQ_DTYPE_F16) return launch_chained(quantize8_kernel<D, TQ_DTYPE_F16>, grid, block, 0, stream, p);
    if (dtype == TQ_DTYPE_BF16) return launch_chained(quantize8_kernel<D, TQ_DTYPE_BF16>, grid, block, 0, stream, p);
    return launch_chained(quantize8_kernel<D, TQ_DTYPE_F32>, grid, block, 0, stream, p);
}

}  // namespace
}  // namespace tq

extern "C" int tq_cache8_page_bytes(int head_dim) {
    return head_dim == 64 || head_dim == 128 ? tq::cache8_page_bytes(head_dim) : TQ_ERR_UNSUPPORTED;
}

extern "C" int tq_quantize8_paged(const void* key, const void* value, int in_dtype, int64_t k_stride_token, int64_t k_stride_head,
                                  int64_t v_stride_token, int64_t v_stride_head, void* cache, int64_t num_blocks, int block_size,
                                  const int64_t* slot_mapping, int64_t n_tokens, int n_kv_heads, int head_dim, int32_t* status,
                                  tq_stream_t stream) {
    using namespace tq;
    if (n_tokens < 0 || n_kv_heads < 0 || num_blocks < 0) return TQ_ERR_ARG;
    if (n_tokens > INT32_MAX || n_kv_heads > 16384 || (head_dim != 64 && head_dim != 128)) return TQ_ERR_UNSUPPORTED;
    if (in_dtype != TQ_DTYPE_F16 && in_dtype != TQ_DTYPE_BF16 && in_dtype != TQ_DTYPE_F32) return TQ_ERR_UNSUPPORTED;
    if (block_size < kPageTokens || block_size % kPageTokens) return TQ_ERR_UNSUPPORTED;
    if (n_tokens == 0 || n_kv_heads == 0 || num_blocks == 0) return TQ_OK;
    if (!key || !value || !cache || !slot_mapping) return TQ_ERR_ARG;
    const int64_t item = in_dtype == TQ_DTYPE_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value) | static_cast<uint64_t>(k_stride_token * item) |
         static_cast<uint64_t>(k_stride_head * item) | static_cast<uint64_t>(v_stride_token * item) |
         static_cast<uint64_t>(v_stride_head * item) | reinterpret_cast<uintptr_t>(cache)) % 16 ||
        reinterpret_cast<uintptr_t>(slot_mapping) % 8)
        return TQ_ERR_ARG;
    Quantize8Params p = {};
    p.key = key; p.value = value; p.cache = static_cast<uint8_t*>(cache); p.slots = slot_mapping; p.status = status;
    p.k_token = k_stride_token; p.k_head = k_stride_head; p.v_token = v_stride_token; p.v_head = v_stride_head;
    p.n_slots = num_blocks * block_size; p.n_tokens = static_cast<int>(n_tokens); p.heads = n_kv_heads;
    p.pages_per_block = block_size / kPageTokens;
    // The rows may be one run each (a decode step) or 16 (a prompt), which the host cannot tell.  Small windows spread single
    // rows over the GPU, large ones leave no block without a run in a prompt; their blocks stay for several, with the next slots asked
    // for ahead.
    p.window = n_tokens <= 512 ? 1 : n_tokens <= 4096 ? 4 : 16;
    const int per_window = p.window == 16 ? 1 : (2 * n_kv_heads + kWarps - 1) / kWarps;
    const int64_t windows = (n_tokens + p.window - 1) / p.window, most = p.window == 16 ? 148 * 4 : windows;
    const dim3 grid(static_cast<unsigned>(windows < most ? windows : most), static_cast<unsigned>(per_window));
    const cudaError_t err = head_dim == 64 ? launch_quantize8<64>(p, in_dtype, grid, stream) : launch_quantize8<128>(p, in_dtype, grid, stream);
    return err == cudaSuccess ? TQ_OK : TQ_ERR_LAUNCH;
}
