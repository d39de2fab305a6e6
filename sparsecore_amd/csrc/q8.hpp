// Optimizer moments in 8 bits: blocks of SLK_Q8_BLOCK elements share one
// float32 scale, the block's largest magnitude. A code is a power of the
// magnitude, so that small values keep digits:
//
//   first moment   q in [-127, 127]:  x = (q/127)·|q/127| · scale
//   second moment  q in [0, 255]:     x = (q/255)^4 · scale
//
// A step of q changes x by the relative 2/q or 4/q; the smallest non-zero
// values are 6.2e-5 and 2.4e-10 of the scale. (A linear code would turn the
// second moment of most elements of a block into 0 and their update into
// m / eps.) A positive second moment never becomes code 0, for the same
// reason. Every operation below is one correctly rounded float32 operation in
// the order written (the build contracts nothing), so codes do not depend on
// the kernel that makes them. A block that holds an infinity or NaN gets a
// non-finite scale and decodes to NaN as a whole: the fault stays visible.
#pragma once

#include "common.hpp"

namespace slk {

constexpr int kQ8Block = SLK_Q8_BLOCK;
static_assert(kQ8Block == 4 * kWave, "four elements a lane: a wave holds one block");

__device__ __forceinline__ float q8_decode_signed(int q, float scale) {
    const float t = static_cast<float>(q) * (1.0f / 127.0f);
    return (t * fabsf(t)) * scale;
}

__device__ __forceinline__ float q8_decode_unsigned(int q, float scale) {
    float t = static_cast<float>(q) * (1.0f / 255.0f);
    t = t * t;
    return (t * t) * scale;
}

// The code that the definition's operations give: one division, one or two
// square roots, correctly rounded (about ten instructions each). Clamped before
// the conversion: a NaN becomes code 0.
__device__ inline float q8_root_signed(float x, float scale) {
    const float a = scale > 0.0f ? fabsf(x) / scale : 0.0f;
    return fminf(fmaxf(rintf(sqrtf(a) * 127.0f), 0.0f), 127.0f);
}
__device__ inline float q8_root_unsigned(float x, float scale) {
    const float a = scale > 0.0f ? fabsf(x) / scale : 0.0f;
    return fminf(fmaxf(rintf(sqrtf(sqrtf(a)) * 255.0f), 0.0f), 255.0f);
}

// The same code from the block's reciprocal and the square root instruction,
// each within an ulp: the value before rounding is off by less than 1e-4 of a
// step (4e-7 of at most 255), so it rounds as the definition's does unless it
// lies within 2e-4 of a tie. Those (4 in 10000, and whatever is not a number in
// [0, 1] of the scale) take the definition's operations. With these alone a
// step of 8-bit AdamW was bound by them: 314 us for 64 million elements.
__device__ __forceinline__ int q8_encode_signed(float x, float scale, float rcp) {
    const float t = __builtin_amdgcn_sqrtf(fabsf(x) * rcp) * 127.0f;
    float q = rintf(t);
    if (!(fabsf(t - q) < 0.4998f) || !(t < 127.01f)) q = q8_root_signed(x, scale);
    return static_cast<int>(copysignf(q, x));
}

__device__ __forceinline__ int q8_encode_unsigned(float x, float scale, float rcp) {
    const float t =
        __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(fabsf(x) * rcp)) * 255.0f;
    float q = rintf(t);
    if (!(fabsf(t - q) < 0.4998f) || !(t < 255.01f)) q = q8_root_unsigned(x, scale);
    if (x > 0.0f) q = fmaxf(q, 1.0f);
    return static_cast<int>(q);
}

// Of 0 or a subnormal scale the instruction gives inf, of one whose reciprocal would be
// subnormal it may give 0: with inf, codes are the definition's.
__device__ __forceinline__ float q8_reciprocal(float scale) {
    return scale < 0x1p126f ? __builtin_amdgcn_rcpf(scale) : INFINITY;
}

// The largest magnitude over the wave's block, four values a lane, or NaN if
// one of them is not finite. Compared as bit patterns: a NaN is above infinity
// there and is kept.
__device__ __forceinline__ float q8_block_max(const float (&x)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(m, o)));
    return __uint_as_float(m < 0x7f800000u ? m : 0x7fc00000u);
}

}  // namespace slk
