// Shared by the forward and backward of slk_norm: a token's features in the
// registers of a team of waves, and sums over the team.
#pragma once

#include "elem.hpp"

namespace slk {

// EPL features a lane, TW waves a team (a wave, or the whole workgroup). VEC:
// lane l holds runs of four consecutive features (one load each); else
// features l, l + lanes, ... (any width, any alignment, LDS without
// conflicts).
template <int EPL, int TW, bool VEC>
struct RowLay {
    static constexpr int kLanes = kWave * TW;
    static __device__ __forceinline__ int at(int q, int l) {
        return VEC ? ((q >> 2) * kLanes + l) * 4 + (q & 3) : q * kLanes + l;
    }
};

// v = features of the row at element `off` (0 past d); VEC needs d % 4 == 0
template <class T, int EPL, int TW, bool VEC>
__device__ __forceinline__ void row_load(const void* p, int64_t off, int d, int l,
                                         float (&v)[EPL]) {
    using Lay = RowLay<EPL, TW, VEC>;
    if (VEC) {
#pragma unroll
        for (int q = 0; q < EPL; q += 4) {
            const int e = Lay::at(q, l);
            if (e < d) {
                T::load4(p, off + e, &v[q]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[q + j] = 0.0f;
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const int e = Lay::at(q, l);
            v[q] = e < d ? T::load(p, off + e) : 0.0f;
        }
    }
}

template <class T, int EPL, int TW, bool VEC>
__device__ __forceinline__ void row_store(void* p, int64_t off, int d, int l,
                                          const float (&v)[EPL]) {
    using Lay = RowLay<EPL, TW, VEC>;
    if (VEC) {
#pragma unroll
        for (int q = 0; q < EPL; q += 4) {
            const int e = Lay::at(q, l);
            if (e < d) T::store4(p, off + e, &v[q]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const int e = Lay::at(q, l);
            if (e < d) T::store(p, off + e, v[q]);
        }
    }
}

// Sums of NV values over the team. With more than one wave, through LDS: red
// holds two buffers of NV x TW floats, used in turn (a wave that writes a
// buffer again has passed the barrier of the sum between, which every wave
// reaches after its reads).
template <int TW, int NV>
struct TeamSum {
    float* red;
    int turn = 0;
    __device__ __forceinline__ void operator()(float (&v)[NV]) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o);
        if constexpr (TW > 1) {
            float* b = red + turn * NV * TW;
            turn ^= 1;
            if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
                for (int k = 0; k < NV; ++k) b[k * TW + (threadIdx.x >> 6)] = v[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float s = b[k * TW];
#pragma unroll
                for (int w = 1; w < TW; ++w) s += b[k * TW + w];
                v[k] = s;
            }
        }
    }
};

// Mean and 1 / sqrt(variance + eps) of a row (mean 0 for RMSNorm): two passes
// over registers, so no cancellation of large means.
template <int EPL, int TW, bool VEC, class Sum>
__device__ __forceinline__ void row_stats(const float (&v)[EPL], int d, int l, bool layer,
                                          float inv_d, float eps, Sum& sum, float& mean,
                                          float& rstd) {
    using Lay = RowLay<EPL, TW, VEC>;
    float s[1] = {0.0f};
    mean = 0.0f;
    if (layer) {
#pragma unroll
        for (int q = 0; q < EPL; ++q) s[0] += v[q];
        sum(s);
        mean = s[0] * inv_d;
        s[0] = 0.0f;
    }
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const float c = Lay::at(q, l) < d ? v[q] - mean : 0.0f;
        s[0] = fmaf(c, c, s[0]);
    }
    sum(s);
    rstd = 1.0f / sqrtf(s[0] * inv_d + eps);
}

// Shape of the row kernels for d features, as f(features a lane, waves a
// team): a wave a token up to 1024, else a workgroup. Eight features of each
// array a lane where a workgroup's 16 waves reach: the backward with a post
// norm and a gate holds some twelve arrays in registers.
constexpr int kNormThreads = 256;

template <class F>
void norm_shape(int d, F&& f) {
    using std::integral_constant;
    if (d <= 512) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (d <= 1024) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (d <= 2048) f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    else if (d <= 4096) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (d <= 8192) f(integral_constant<int, 8>{}, integral_constant<int, 16>{});
    else f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
}

int validate_norm(const slk_norm* a, const char* who, bool backward);

inline bool norm_vec(const slk_norm* a, std::initializer_list<const void*> ps) {
    if (a->d % 4 != 0) return false;
    for (const void* p : ps)
        if (p != nullptr && !aligned_to(p, a->dtype == SLK_F32 ? 16 : 8)) return false;
    return true;
}

// Tokens of a workgroup's tile where an array is feature-major, and the LDS
// pitch of a feature's tokens (odd: a wave that walks the features of one
// token, as one that walks tokens, meets every bank once).
constexpr int kTileWaves = 8;
constexpr int kTileThreads = kTileWaves * kWave;

// Copies a feature-major d x n array's columns [n0, n0 + TT) into LDS, and back.
template <class T, int TT>
__device__ __forceinline__ void tile_load(const void* src, int64_t n, int d, int64_t n0,
                                          float* tile) {
    const int t = threadIdx.x % TT;
    const bool in = n0 + t < n;
    for (int e0 = threadIdx.x / TT; e0 < d; e0 += 8 * (kTileThreads / TT)) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = e0 + j * (kTileThreads / TT);
            v[j] = in && e < d ? T::load(src, static_cast<int64_t>(e) * n + n0 + t) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = e0 + j * (kTileThreads / TT);
            if (e < d) tile[e * (TT + 1) + t] = v[j];
        }
    }
}

template <class T, int TT>
__device__ __forceinline__ void tile_store(void* dst, int64_t n, int d, int64_t n0,
                                           const float* tile) {
    const int t = threadIdx.x % TT;
    if (n0 + t >= n) return;
    for (int e = threadIdx.x / TT; e < d; e += kTileThreads / TT)
        T::store(dst, static_cast<int64_t>(e) * n + n0 + t, tile[e * (TT + 1) + t]);
}

template <int EPL, int TT>
__device__ __forceinline__ void tile_row_load(const float* tile, int t, int d, int l,
                                              float (&v)[EPL]) {
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = q * kWave + l;
        v[q] = e < d ? tile[e * (TT + 1) + t] : 0.0f;
    }
}

template <int EPL, int TT>
__device__ __forceinline__ void tile_row_store(float* tile, int t, int d, int l,
                                               const float (&v)[EPL]) {
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = q * kWave + l;
        if (e < d) tile[e * (TT + 1) + t] = v[q];
    }
}

}  // namespace slk
