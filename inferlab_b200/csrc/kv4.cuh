// kv4.cuh - the packed 4-bit pool: what a code stands for and where it lies.
//
// Every 64 dims of one token's K or V row of one kv-head share a pair of f16
// numbers (scale, zero); a code c in 0..15 stands for zero + (c - 8) * scale.
// A row is quantised from values x already rounded to the pool's 16-bit row
// type:
//   scale = f16((max - min) / 15)     zero = f16(min + 8 * scale)
//   c = clamp(rint((x - zero) * (1 / scale)) + 8, 0, 15), 8 where scale is 0.
// Codes counted from 8 keep sum p (c - 8) a sum of either sign, so that the
// fp32 accumulators of a long, flat softmax do not grow far beyond the output.
//
// One arena [num_blocks][kv_heads][block_tokens / 16][tile]. A tile is 16
// tokens of one kv-head in one contiguous run, so one bulk copy moves it:
//   key codes   [16][D / 2] bytes, key pairs   [16][D / 64] (scale, zero),
//   value codes [16][D / 2] bytes, value pairs [16][D / 64] (scale, zero).
// D = 128: 2304 bytes (144 a token against 512 in 16 bits), D = 64: 1152.
//
// A code row is made of 32-bit words of 8 consecutive dims (dim 8 w + n in
// bits 4n..4n+3). The words are ordered for the attention's mma fragments, so
// that a lane reads its part of a row with one load:
//   keys:   lane t of four holds, for every 32 dims, dims 8t .. 8t+7;
//           word (w, t) (dims 32 w + 8 t ..) lies at t * D / 8 + 4 w bytes.
//   values: lane g of eight holds, for every 64 dims, dims 8g .. 8g+7;
//           word (w, g) (dims 64 w + 8 g ..) lies at g' * D / 16 + 4 w bytes,
//           g' = g, but g ^ 4 in tokens 2, 3 of every four when D is 128: four
//           token rows read by four lanes then fall on different banks.
#pragma once

#include "common.cuh"

namespace ilb {
namespace kv4 {

constexpr int kGroup = 64;       // dims that share a (scale, zero) pair
constexpr int kTileTokens = 16;

__host__ __device__ constexpr int code_bytes(int d) { return kTileTokens * (d / 2); }
__host__ __device__ constexpr int pair_bytes(int d) { return kTileTokens * (d / kGroup) * 4; }
__host__ __device__ constexpr int half_tile_bytes(int d) { return code_bytes(d) + pair_bytes(d); }
__host__ __device__ constexpr int tile_bytes(int d) { return 2 * half_tile_bytes(d); }

// Byte of the word that holds dims 8 unit .. 8 unit + 7 of token slot `t`.
__device__ __forceinline__ int key_word(int d, int t, int unit) {
    return t * (d / 2) + (unit & 3) * (d / 8) + (unit >> 2) * 4;
}
__device__ __forceinline__ int value_word(int d, int t, int unit) {
    const int chunk = (unit & 7) ^ (d == 128 ? ((t >> 1) & 1) * 4 : 0);
    return half_tile_bytes(d) + t * (d / 2) + chunk * (d / 16) + (unit >> 3) * 4;
}
// Byte of the (scale, zero) pair of group `g` of token slot `t`; value = 0 / 1.
__device__ __forceinline__ int pair_at(int d, int t, int g, int value) {
    return value * half_tile_bytes(d) + code_bytes(d) + (t * (d / kGroup) + g) * 4;
}

__device__ __forceinline__ float2 load_pair(const unsigned char* tile, int at) {
    return __half22float2(*reinterpret_cast<const __half2*>(tile + at));
}

// Two fp32 lanes an instruction, each rounded as the scalar would be. A sum of
// such products takes scalar additions: ptxas makes a mul.f32x2 and an
// add.f32x2 one fma, explicit rounding or not.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    std::uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pack_f32x2(a.x, a.y)), "l"(pack_f32x2(b.x, b.y)));
    return make_float2(low_f32(d), high_f32(d));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    std::uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pack_f32x2(a.x, a.y)), "l"(pack_f32x2(b.x, b.y)));
    return make_float2(low_f32(d), high_f32(d));
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return add2(a, make_float2(-b.x, -b.y)); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    std::uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pack_f32x2(a.x, a.y)), "l"(pack_f32x2(b.x, b.y)), "l"(pack_f32x2(c.x, c.y)));
    return make_float2(low_f32(d), high_f32(d));
}
// Maximum of three that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The values of a word's eight codes, as code_value.
__device__ __forceinline__ void code_values(std::uint32_t word, float2 pair, float (&x)[8]) {
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
        const float2 c = make_float2(__uint_as_float(((word >> (4 * n)) & 15u) | 0x4b000000u),
                                     __uint_as_float(((word >> (4 * n + 4)) & 15u) | 0x4b000000u));
        const float2 v = mul2(add2(c, make_float2(-8388616.0f, -8388616.0f)), make_float2(pair.x, pair.x));
        x[n] = __fadd_rn(v.x, pair.y), x[n + 1] = __fadd_rn(v.y, pair.y);
    }
}

// A code's value, fp32 with one rounding per operation.
__device__ __forceinline__ float code_value(std::uint32_t word, int n, float2 pair) {
    // 2^23 + c by its bits, less 2^23 + 8: exact, and no conversion instruction.
    const float c = __uint_as_float(((word >> (4 * n)) & 15u) | 0x4b000000u) - 8388616.0f;
    return __fadd_rn(__fmul_rn(c, pair.x), pair.y);
}

// Quantises the 8 dims of this lane's unit; the 8 lanes of an aligned octet
// hold the 64 dims of one group. Returns the word of codes and the pair;
// `bad` reports a non-finite value or a pair outside f16.
__device__ __forceinline__ std::uint32_t quantise(const float (&x)[8], __half2& pair, bool& bad) {
    // A NaN survives into the range and so into the scale; an infinity is one.
    float high = max3_nan(max3_nan(x[0], x[1], x[2]), x[3], max3_nan(x[4], x[5], max3_nan(x[6], x[7], x[7])));
    float low = -max3_nan(max3_nan(-x[0], -x[1], -x[2]), -x[3], max3_nan(-x[4], -x[5], max3_nan(-x[6], -x[7], -x[7])));
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
        const float other_low = __shfl_xor_sync(0xffffffffu, low, off), other_high = __shfl_xor_sync(0xffffffffu, high, off);
        low = fminf(low, other_low);
        high = max3_nan(high, other_high, other_high);
    }
    // (high - low) / 15, correctly rounded: a product with the rounded
    // reciprocal and one correction by the exact remainder (Markstein). Where
    // the remainder would underflow the scale is 0 in f16 anyway.
    const float range = __fsub_rn(high, low);
    const float guess = __fmul_rn(range, 0.06666667014360428f);
    const float quotient = __fmaf_rn(__fmaf_rn(-15.0f, guess, range), 0.06666667014360428f, guess);
    const __half scale_h = __float2half_rn(quotient);
    const float scale = __half2float(scale_h);
    const __half zero_h = __float2half_rn(__fadd_rn(low, 8.0f * scale));
    const float zero = __half2float(zero_h);
    bad = !isfinite(scale) || !isfinite(zero);
    pair = __halves2half2(scale_h, zero_h);
    const float inverse = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
    // Steps from the zero, clamped to -8..7, to the nearest (ties to even) by
    // adding 1.5 2^23, then counted from -8: all exact, so four codes are one
    // fp32 number below 2^16.
    float part[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float c[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float2 t = mul2(sub2(make_float2(x[4 * half + i], x[4 * half + i + 1]), make_float2(zero, zero)), make_float2(inverse, inverse));
            t = make_float2(fminf(fmaxf(t.x, -8.0f), 7.0f), fminf(fmaxf(t.y, -8.0f), 7.0f));
            t = sub2(add2(t, make_float2(12582912.0f, 12582912.0f)), make_float2(12582904.0f, 12582904.0f));
            c[i] = t.x, c[i + 1] = t.y;
        }
        part[half] = fmaf(fmaf(fmaf(c[3], 16.0f, c[2]), 16.0f, c[1]), 16.0f, c[0]);
    }
    return static_cast<std::uint32_t>(__float2int_rn(part[0])) | static_cast<std::uint32_t>(__float2int_rn(part[1])) << 16;
}

}  // namespace kv4
}  // namespace ilb
