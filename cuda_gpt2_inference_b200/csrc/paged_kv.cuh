// paged_kv.cuh -- number format of the 4-bit KV cache, shared by the append,
// read-back and attention kernels.
#pragma once

#include "common.cuh"

namespace gpt2b {

constexpr int kW4Group = 64;  // channels that share a step and a low end
constexpr int kW4Tile = 16;   // block sizes are multiples of this, so a 16-row tile lies in one block
constexpr int kTableMaxRequests = 4096;

// of BF16 pairs; NaN wins, so one NaN in a group reaches its ends
__device__ __forceinline__ uint32_t bf16x2_min_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ uint32_t bf16x2_max_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// FP32 operations that keep subnormals, which the build's fast arithmetic takes as 0: BF16 inputs may be subnormal,
// and beside a step of 2^-120 they are up to 2^-6 of it.
__device__ __forceinline__ float mul_sub(float a, float b) {
    float r;
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float fma_sub(float a, float b, float c) {
    float r;
    asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 16 channels (8 BF16 pairs u) of a group with ends [lo, hi] (minus_hi: a negation would lose a subnormal) -> two
// words of codes; meta = step | low end << 16 (BF16 bits).  step = bf16(hi/15 - lo/15): each product and the difference rounded on its own, so that a
// range beyond FP32's does not overflow.  A step below 2^-120 is held as 0 (codes 0): the division below
// then never meets a subnormal.  The code is taken from halves, x/2 - lo/2 over step/2, for the same reason
// of range.  The step is rounded to nearest, not up: the top code then misses hi by at most 15 * 2^-8 of a
// step, and no quotient reaches 15.5.  A group with a NaN or an infinity is held as NaN.
//
// Each code is the quotient rounded to the nearest whole number, ties to even, where a quotient within 2^-17 of a
// half counts as one.  The quotient is a product with an approximate reciprocal, off by 2^-19 at most, rounded to
// a grid of 2^-16 on its way: a tie (frequent with BF16 values over a step of few bits) is one again there.
__device__ __forceinline__ uint2 w4_encode16(const uint32_t* u, float lo, float minus_hi, uint32_t& meta) {
    const float c = 1.0f / 15.0f;
    if (!(fabsf(lo) < INFINITY && fabsf(minus_hi) < INFINITY)) {
        meta = 0x7fc07fc0u;
        return make_uint2(0u, 0u);
    }
    float t = fma_sub(mul_sub(lo, c), -1.0f, mul_sub(minus_hi, -c));  // (the product with -1 is exact)
    if (t < 0x1p-120f) t = 0.0f;
    const uint32_t sbits = __bfloat16_as_ushort(__float2bfloat16_rn(t));
    meta = sbits | (__float_as_uint(lo) & 0xffff0000u);  // lo is a BF16 value
    if (sbits == 0) return make_uint2(0u, 0u);
    const float half = 0.5f * __uint_as_float(sbits << 16), nlo = mul_sub(lo, -0.5f), inv = __fdividef(1.0f, half);
    constexpr float kGrid = 192.0f;        // added, it rounds 0 .. 15.5 to multiples of 2^-16
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: added, it rounds to a whole number
    uint32_t word[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float code[8], h[2];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t p = u[4 * i + k / 2];
            const float d = fma_sub(k & 1 ? bf16hi(p) : bf16lo(p), 0.5f, nlo);  // the product is exact
            code[k] = __fsub_rn(__fadd_rn(fmaf(d, inv, kGrid), kRound - kGrid), kRound);
        }
        // four codes to a 16-bit whole number on the FMA units, its bits under the exponent of 2^23
#pragma unroll
        for (int k = 0; k < 2; k++)
            h[k] = fmaf(code[4 * k + 3], 4096.0f, fmaf(code[4 * k + 2], 256.0f, fmaf(code[4 * k + 1], 16.0f, code[4 * k]))) +
                   8388608.0f;
        word[i] = __byte_perm(__float_as_uint(h[0]), __float_as_uint(h[1]), 0x5410);
    }
    return make_uint2(word[0], word[1]);
}

// The 8 channels of a word as FP32: code * step + low end, one rounding (subnormals kept).  Nibble k of a half, masked in place
// under the exponent of 2^23, reads 2^23 + code * 16^k; one exact multiply-add leaves the code.
__device__ __forceinline__ void w4_values(uint32_t word, uint32_t meta, float* x) {
    const float s = __uint_as_float(meta << 16), lo = __uint_as_float(meta & 0xffff0000u);
    const float down[4] = {1.0f, 0x1p-4f, 0x1p-8f, 0x1p-12f};
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const uint32_t h = k < 4 ? word : word >> 16;
        const float f = __uint_as_float((h & (15u << (4 * (k & 3)))) | 0x4b000000u);
        x[k] = fma_sub(fmaf(f, down[k & 3], -8388608.0f * down[k & 3]), s, lo);
    }
}

}  // namespace gpt2b
