// Page layout of the 8-bit cache and its number format, shared by the kernels that write and read it.
//
// A page holds 16 tokens of one KV head: K codes [16][D], V codes [16][D] (e4m3, one byte each), then two fp32 scales (K, V) and
// 24 bytes that nothing reads, so that pages are whole 32-byte sectors.  A value is code * scale; a scale is a power of two.
#pragma once

#include "tq_common.cuh"

namespace tq {

constexpr int kMinExponent = -100;      // of a scale: smaller values are zero, and 2^100 * value stays finite in fp32
constexpr int kMaxExponent = 120;       // 448 * 2^120 is beyond every finite fp32 value

__host__ __device__ constexpr int cache8_page_bytes(int head_dim) { return 2 * kPageTokens * head_dim + 32; }
__host__ __device__ constexpr int cache8_scale_off(int head_dim) { return 2 * kPageTokens * head_dim; }

// Smallest e with amax <= 448 * 2^e.  448 = 1.75 * 2^8, so a mantissa above 1.75 carries into the next exponent.
__host__ __device__ __forceinline__ int scale_exponent_of_bits(uint32_t amax_bits) {
    const int e = static_cast<int>((amax_bits + 0x1fffffu) >> 23) - 127 - 8;
    return e < kMinExponent ? kMinExponent : e > kMaxExponent ? kMaxExponent : e;
}

// The exponent of a scale as a page holds it; anything that is no scale (a page that nothing was written to) counts as the least.
__host__ __device__ __forceinline__ int exponent_of_scale_bits(uint32_t scale_bits) {
    const int e = static_cast<int>(scale_bits >> 23) - 127;         // a sign bit makes e large: beyond the maximum
    return e < kMinExponent || e > kMaxExponent ? kMinExponent : e;
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }   // |e| <= 126; -127 makes zero

// two floats -> two e4m3 codes, lo in bits 0..7; nearest even, saturating (infinities too), NaN stays one
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// two e4m3 codes (bits 0..15) -> half2, exact
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(codes)));
    return h2;
}

}  // namespace tq
