// paged_kv.cuh -- number format of the 4-bit KV cache, shared by the append,
// read-back and attention kernels.
#pragma once

#include "common.cuh"

namespace gpt2b {

constexpr int kW4Group = 64;  // channels that share a step and a low end
constexpr int kW4Tile = 16;   // block sizes are multiples of this, so a 16-row tile lies in one block
constexpr int kTableMaxRequests = 4096;

// 8 channels of a group with ends [lo, hi] -> one word of codes; meta = step | low end << 16 (BF16 bits).
// step = bf16(hi/15 - lo/15): each product and the difference rounded on its own, so that a range
// beyond FP32's does not overflow.  A step below 2^-120 is held as 0 (codes 0): the division below
// then never meets a subnormal.  The code is taken from halves for the same reason of range.
// The step is rounded to nearest, not up: the top code then misses hi by at most 15 * 2^-9 of a step.
// A group with a NaN or an infinity (fin false) is held as NaN.
__device__ __forceinline__ uint32_t w4_encode8(const float* x, float lo, float hi, bool fin, uint32_t& meta) {
    const float c = 1.0f / 15.0f;
    float t = __fsub_rn(__fmul_rn(hi, c), __fmul_rn(lo, c));
    if (t < 7.52316385e-37f) t = 0.0f;  // 2^-120
    const uint32_t sbits = __bfloat16_as_ushort(__float2bfloat16_rn(t));
    const float half = 0.5f * __uint_as_float(sbits << 16);
    if (!fin) {
        meta = 0x7fc07fc0u;
        return 0u;
    }
    meta = sbits | (__float_as_uint(lo) & 0xffff0000u);  // lo is a BF16 value
    uint32_t word = 0u;
    if (half > 0.0f) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d = __fsub_rn(__fmul_rn(x[k], 0.5f), __fmul_rn(lo, 0.5f));
            const float q = fminf(rintf(__fdiv_rn(d, half)), 15.0f);
            word |= (uint32_t)(int)q << (4 * k);
        }
    }
    return word;
}

// Channel j (0..7) of a word as FP32: code * step + low end, one rounding.
__device__ __forceinline__ float w4_value(uint32_t word, uint32_t meta, int j) {
    return fmaf((float)((word >> (4 * j)) & 15u), __uint_as_float(meta << 16), __uint_as_float(meta & 0xffff0000u));
}

}  // namespace gpt2b
