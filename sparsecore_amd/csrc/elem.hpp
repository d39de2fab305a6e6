// Elements of dense arrays by type: one, or four consecutive ones in one load.
// Arithmetic on them is float32 throughout.
#pragma once

#include "common.hpp"

namespace slk {

struct F32 {
    static constexpr int kBytes = 4;
    static __device__ __forceinline__ float load(const void* p, int64_t i) {
        return static_cast<const float*>(p)[i];
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
        static_cast<float*>(p)[i] = v;
    }
    static __device__ __forceinline__ void load4(const void* p, int64_t i, float* v) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j];
    }
    static __device__ __forceinline__ void store4(void* p, int64_t i, const float* v) {
        f32x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = v[j];
        *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = x;
    }
};

struct BF16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ float load(const void* p, int64_t i) {
        return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
        static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
    }
    static __device__ __forceinline__ void load4(const void* p, int64_t i, float* v) {
        const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        v[0] = bf16_to_f32(x.x & 0xffffu);
        v[1] = bf16_to_f32(x.x >> 16);
        v[2] = bf16_to_f32(x.y & 0xffffu);
        v[3] = bf16_to_f32(x.y >> 16);
    }
    static __device__ __forceinline__ void store4(void* p, int64_t i, const float* v) {
        uint2 x;
        x.x = f32_to_bf16(v[0]) | (static_cast<uint32_t>(f32_to_bf16(v[1])) << 16);
        x.y = f32_to_bf16(v[2]) | (static_cast<uint32_t>(f32_to_bf16(v[3])) << 16);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = x;
    }
};

inline bool aligned_to(const void* p, uintptr_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace slk
