// Rotary positions of query and key heads, in one pass over both.
//
//   half layout         y[i] = x[i] c_i - x[i + R/2] s_i,   y[i + R/2] = x[i + R/2] c_i + x[i] s_i      (0 <= i < R/2)
//   interleaved layout  the same on the pairs (x[2i], x[2i + 1])
//
// with R = rotary_dim <= head_dim, values from R on copied, and (c_i, s_i) the row of the fp32 table that the token's position
// names; `inverse` turns the other way (s -> -s).  Arithmetic in fp32, one rounding.
//
// Bound: HBM, each value read and written once.  A thread owns one vector of a head, with its partners: both halves of the
// pairs for the half layout, so that rotating in place is safe.  It keeps its cosines and sines in registers and walks over
// heads of the same token: the table (fp32, shared by all heads) would otherwise be twice the traffic of the rows themselves.
#include "tq_common.cuh"

namespace tq {
namespace {

struct RotaryParams {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    const void* positions;
    const float* table;
    int32_t* status;
    int64_t q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;   // strides in elements
    int64_t table_rows;
    int rows, q_heads, heads;       // heads = q_heads + kv heads
    int rotary_dim;
    int units, pair_units;          // vectors of a head that a thread owns one of; those with a rotation
    int slots, rows_per_block;      // heads at a time, tokens at a time
    int wide_positions, inverse;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};
// Rows of a large call pass through once: marked so, they do not push one another's lines out of L2 half written (16411 rows of 40
// heads in bf16: 77.8 us without, 55.4 with).
template <bool ONCE, typename V>
__device__ __forceinline__ V load_row(const V* p) {
    V v;
    if constexpr (ONCE && sizeof(V) == 16) *reinterpret_cast<uint4*>(&v) = __ldcs(reinterpret_cast<const uint4*>(p));
    else v = *p;
    return v;
}
template <bool ONCE, typename V>
__device__ __forceinline__ void store_row(V* p, const V& v) {
    if constexpr (ONCE && sizeof(V) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
    else *p = v;
}
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }

// N: elements of a vector.  ITER: heads per thread.
template <typename T, int N, bool INTERLEAVED, int ITER>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
    pdl_wait();
    pdl_release_if_small();
    constexpr int kPairs = INTERLEAVED ? N / 2 : N;
    const int per_row = p.units * p.slots;
    const int local = threadIdx.x / per_row, rest = threadIdx.x - local * per_row;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * p.rows_per_block + local;
    if (local >= p.rows_per_block || row >= p.rows) return;
    const int slot = rest / p.units, unit = rest - slot * p.units;
    const bool turned = unit < p.pair_units;
    const int half = p.rotary_dim / 2;
    const int first = turned ? unit * N : p.rotary_dim + (unit - p.pair_units) * N;   // element of the head

    Vec<T, N> x[ITER], y[ITER];
    const T* in[ITER];
    T* out[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int h = (blockIdx.y * ITER + i) * p.slots + slot;
        out[i] = nullptr;
        if (h < p.heads) {
            const bool is_q = h < p.q_heads;
            const int hh = is_q ? h : h - p.q_heads;
            in[i] = static_cast<const T*>(is_q ? p.q : p.k) + row * (is_q ? p.q_row : p.k_row) + hh * (is_q ? p.q_head : p.k_head) + first;
            out[i] = static_cast<T*>(is_q ? p.q_out : p.k_out) + row * (is_q ? p.qo_row : p.ko_row) + hh * (is_q ? p.qo_head : p.ko_head) + first;
            x[i] = load_row<(ITER > 1)>(reinterpret_cast<const Vec<T, N>*>(in[i]));
            if (!INTERLEAVED && turned) y[i] = load_row<(ITER > 1)>(reinterpret_cast<const Vec<T, N>*>(in[i] + half));
        }
    }
    if (!turned) {
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if (out[i]) store_row<(ITER > 1)>(reinterpret_cast<Vec<T, N>*>(out[i]), x[i]);
        return;
    }
    int64_t pos = p.wide_positions ? static_cast<const int64_t*>(p.positions)[row] : static_cast<const int32_t*>(p.positions)[row];
    if (pos < 0 || pos >= p.table_rows) {
        if (p.status && unit == 0 && slot == 0 && blockIdx.y == 0) atomicOr(p.status, TQ_STATUS_BAD_POSITION);
        pos = pos < 0 ? 0 : p.table_rows - 1;
    }
    const float* t = p.table + pos * p.rotary_dim + (INTERLEAVED ? first / 2 : first);
    float c[kPairs], s[kPairs];
    if constexpr (kPairs % 4 == 0) {
#pragma unroll
        for (int j = 0; j < kPairs; j += 4) {
            const float4 a = *reinterpret_cast<const float4*>(t + j), b = *reinterpret_cast<const float4*>(t + half + j);
            c[j] = a.x; c[j + 1] = a.y; c[j + 2] = a.z; c[j + 3] = a.w;
            s[j] = b.x; s[j + 1] = b.y; s[j + 2] = b.z; s[j + 3] = b.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            c[j] = t[j];
            s[j] = t[half + j];
        }
    }
    if (p.inverse) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) s[j] = -s[j];
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (!out[i]) continue;
        Vec<T, N> a, b;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            const float u = to_float(INTERLEAVED ? x[i].v[2 * j] : x[i].v[j]), w = to_float(INTERLEAVED ? x[i].v[2 * j + 1] : y[i].v[j]);
            const T ru = from_float<T>(u * c[j] - w * s[j]), rw = from_float<T>(w * c[j] + u * s[j]);
            if (INTERLEAVED) {
                a.v[2 * j] = ru;
                a.v[2 * j + 1] = rw;
            } else {
                a.v[j] = ru;
                b.v[j] = rw;
            }
        }
        store_row<(ITER > 1)>(reinterpret_cast<Vec<T, N>*>(out[i]), a);
        if (!INTERLEAVED) store_row<(ITER > 1)>(reinterpret_cast<Vec<T, N>*>(out[i] + half), b);
    }
}

template <typename T, int N, bool INTERLEAVED>
cudaError_t launch_rotary(RotaryParams p, int head_dim, cudaStream_t stream) {
    p.pair_units = p.rotary_dim / N / (INTERLEAVED ? 1 : 2);
    p.units = p.pair_units + (head_dim - p.rotary_dim) / N;
    // Few tokens: a head per thread and many blocks, the call is a chain of load latencies.  Many: four vectors per thread in flight -
    // four heads, or two of the half layout - which share the table's.  (Half layout, 16000 rows of 40 heads in bf16: 58.6 us with two
    // heads, 72.9 with four; interleaved, half of each head: 55.4 with four, 76 with two.)
    constexpr int kMany = INTERLEAVED ? 4 : 2;
    const bool few = static_cast<int64_t>(p.rows) * p.heads * p.units <= 148 * 1024;
    const int iter = few ? 1 : kMany;
    p.slots = (p.heads + iter - 1) / iter;
    if (p.slots > 256 / p.units) p.slots = 256 / p.units;
    p.rows_per_block = few ? 1 : 256 / (p.slots * p.units);
    const int threads = (p.slots * p.units * p.rows_per_block + 31) / 32 * 32;
    const dim3 grid(static_cast<unsigned>((p.rows + p.rows_per_block - 1) / p.rows_per_block),
                    static_cast<unsigned>((p.heads + p.slots * iter - 1) / (p.slots * iter)));
    return few ? launch_chained(rotary_kernel<T, N, INTERLEAVED, 1>, grid, dim3(threads), 0, stream, p)
               : launch_chained(rotary_kernel<T, N, INTERLEAVED, kMany>, grid, dim3(threads), 0, stream, p);
}

template <typename T>
cudaError_t launch_type(const RotaryParams& p, int head_dim, int n, int interleaved, cudaStream_t stream) {
    if (interleaved) {
        if (n * sizeof(T) == 16) return launch_rotary<T, 16 / sizeof(T), true>(p, head_dim, stream);
        if (n == 4) return launch_rotary<T, 4, true>(p, head_dim, stream);
        return launch_rotary<T, 2, true>(p, head_dim, stream);
    }
    if (n * sizeof(T) == 16) return launch_rotary<T, 16 / sizeof(T), false>(p, head_dim, stream);
    if (n == 4) return launch_rotary<T, 4, false>(p, head_dim, stream);
    if (n == 2) return launch_rotary<T, 2, false>(p, head_dim, stream);
    return launch_rotary<T, 1, false>(p, head_dim, stream);
}

}  // namespace
}  // namespace tq

extern "C" int tq_rotary(const void* q, const void* k, void* q_out, void* k_out, int dtype, const int64_t* strides, const void* positions,
                         int wide_positions, const float* table, int64_t table_rows, int64_t rows, int num_q_heads, int num_kv_heads, int head_dim,
                         int rotary_dim, int interleaved, int inverse, int32_t* status, tq_stream_t stream) {
    using namespace tq;
    if (rows < 0 || rows > INT32_MAX || num_q_heads < 0 || num_kv_heads < 0 || table_rows < 1 || !strides) return TQ_ERR_ARG;
    if (dtype != TQ_DTYPE_F16 && dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F32) return TQ_ERR_UNSUPPORTED;
    if (head_dim < 2 || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim) return TQ_ERR_ARG;
    const int64_t heads = static_cast<int64_t>(num_q_heads) + num_kv_heads;
    if (rows == 0 || heads == 0) return TQ_OK;
    if (heads > 16384) return TQ_ERR_UNSUPPORTED;
    if (!positions || !table || (num_q_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out))) return TQ_ERR_ARG;
    const int item = dtype == TQ_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(positions) % (wide_positions ? 8 : 4) || reinterpret_cast<uintptr_t>(table) % 4) return TQ_ERR_ARG;
    // The widest vector that every row, head and part of a head starts on.
    uint64_t bits = static_cast<uint64_t>(interleaved ? rotary_dim : rotary_dim / 2) * item | static_cast<uint64_t>(head_dim - rotary_dim) * item;
    if (num_q_heads)
        bits |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | static_cast<uint64_t>(strides[0] * item) |
                static_cast<uint64_t>(strides[1] * item) | static_cast<uint64_t>(strides[4] * item) | static_cast<uint64_t>(strides[5] * item);
    if (num_kv_heads)
        bits |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) | static_cast<uint64_t>(strides[2] * item) |
                static_cast<uint64_t>(strides[3] * item) | static_cast<uint64_t>(strides[6] * item) | static_cast<uint64_t>(strides[7] * item);
    if (bits % item) return TQ_ERR_ARG;
    int n = 16 / item;
    while (n > 1 && bits % (static_cast<uint64_t>(n) * item)) n /= 2;
    // The table is read four pairs at a time where a vector holds four; its rows then start on 16 bytes.
    const auto pairs = [&](int m) { return interleaved ? m / 2 : m; };
    while (n > 1 && pairs(n) % 4 == 0 && (reinterpret_cast<uintptr_t>(table) % 16 || (rotary_dim / 2) % 4)) n /= 2;
    if (interleaved && n < 2) return TQ_ERR_ARG;                        // a pair does not start on its own size
    const int units = (interleaved ? rotary_dim / n : rotary_dim / 2 / n) + (head_dim - rotary_dim) / n;
    if (units > 256) return TQ_ERR_UNSUPPORTED;
    RotaryParams p = {};
    p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out; p.positions = positions; p.table = table; p.status = status;
    p.q_row = strides[0]; p.q_head = strides[1]; p.k_row = strides[2]; p.k_head = strides[3];
    p.qo_row = strides[4]; p.qo_head = strides[5]; p.ko_row = strides[6]; p.ko_head = strides[7];
    p.table_rows = table_rows; p.rows = static_cast<int>(rows); p.q_heads = num_q_heads; p.heads = static_cast<int>(heads);
    p.rotary_dim = rotary_dim; p.wide_positions = wide_positions; p.inverse = inverse;
    cudaError_t err;
    if (dtype == TQ_DTYPE_F16) err = launch_type<__half>(p, head_dim, n, interleaved, stream);
    else if (dtype == TQ_DTYPE_BF16) err = launch_type<__nv_bfloat16>(p, head_dim, n, interleaved, stream);
    else err = launch_type<float>(p, head_dim, n, interleaved, stream);
    return err == cudaSuccess ? TQ_OK : TQ_ERR_LAUNCH;
}
