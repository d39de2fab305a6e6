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

// The sum over a wave, in every lane: cross-lane adds inside rows of 16 lanes,
// then across rows towards lane 63 (six vector instructions, where shuffles
// through LDS wait six times).
__device__ __forceinline__ float wave_sum(float x) {
    auto add = [&](auto ctrl, auto rows) {
        constexpr int C = decltype(ctrl)::value, R = decltype(rows)::value;
        x += __int_as_float(
            __builtin_amdgcn_update_dpp(0, __float_as_int(x), C, R, 0xf, true));
    };
    using std::integral_constant;
    add(integral_constant<int, 0xB1>{}, integral_constant<int, 0xf>{});   // lane ^ 1
    add(integral_constant<int, 0x4E>{}, integral_constant<int, 0xf>{});   // lane ^ 2
    add(integral_constant<int, 0x141>{}, integral_constant<int, 0xf>{});  // half row mirrored
    add(integral_constant<int, 0x140>{}, integral_constant<int, 0xf>{});  // row mirrored
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // rows 0, 2 to 1, 3
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // lane 31 to rows 2, 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
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
        for (int k = 0; k < NV; ++k) v[k] = wave_sum(v[k]);
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
                f32x4 s = *reinterpret_cast<const f32x4*>(b + k * TW);
#pragma unroll
                for (int w = 4; w < TW; w += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(b + k * TW + w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[j] += x[j];
                }
                v[k] = (s[0] + s[1]) + (s[2] + s[3]);
            }
        }
    }
};

// A row's features as they are in memory (VEC layout): fetched ahead at the
// cost of their own registers, converted when used.
template <class T, int EPL, int TW>
struct RawRow {
    using Piece = std::conditional_t<T::kBytes == 4, f32x4, uint2>;
    Piece p[EPL / 4];
    __device__ __forceinline__ void load(const void* from, int64_t off, int d, int l) {
#pragma unroll
        for (int q = 0; q < EPL / 4; ++q) {
            const int e = RowLay<EPL, TW, true>::at(4 * q, l);
            if (e < d) {
                p[q] = *reinterpret_cast<const Piece*>(static_cast<const char*>(from) +
                                                       (off + e) * T::kBytes);
            } else {
                p[q] = Piece{};
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[EPL]) const {
#pragma unroll
        for (int q = 0; q < EPL / 4; ++q) {
            if constexpr (T::kBytes == 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * q + j] = p[q][j];
            } else {
                v[4 * q] = bf16_to_f32(p[q].x & 0xffffu);
                v[4 * q + 1] = __uint_as_float(p[q].x & 0xffff0000u);
                v[4 * q + 2] = bf16_to_f32(p[q].y & 0xffffu);
                v[4 * q + 3] = __uint_as_float(p[q].y & 0xffff0000u);
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
// team): a wave a token up to 1024, else a workgroup. The backward with a post
// norm and a gate holds some twelve arrays in registers, which 16 features a
// lane make 256 of: eight waves at most then, so 16 only above 8192.
constexpr int kNormThreads = 256;

template <class F>
void norm_shape(int d, F&& f) {
    using std::integral_constant;
    if (d <= 512) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (d <= 1024) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (d <= 2048) f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    else if (d <= 4096) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (d <= 8192) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
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
constexpr int64_t kTileMinGroups = 512;

// The tile's row of feature e: lanes that hold runs of four features (VEC) then
// walk consecutive rows, an odd number of banks apart.
__device__ __forceinline__ int tile_row(int e, int quarter) {
    return (e & 3) * quarter + (e >> 2);
}
__host__ __device__ inline int tile_quarter(int64_t d) { return static_cast<int>((d + 3) / 4); }

// Copies a feature-major d x n array's columns [n0, n0 + TT) into LDS, and back.
// bfloat16 columns go two tokens a lane (pairs: n is even and the array is
// 4-byte aligned), or a row of the tile would be 2 TT bytes of 2-byte accesses.
template <class T, int TT>
__device__ __forceinline__ void tile_load(const void* src, int64_t n, int d, int64_t n0,
                                          bool pairs, float* tile) {
    const int quarter = tile_quarter(d);
    if (T::kBytes == 2 && pairs) {
        constexpr int kCols = TT / 2, kRows = kTileThreads / kCols;
        const int t = 2 * (threadIdx.x % kCols);
        const bool in = n0 + t < n;
        const uint16_t* s = static_cast<const uint16_t*>(src);
        for (int e0 = threadIdx.x / kCols; e0 < d; e0 += 4 * kRows) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = e0 + j * kRows;
                v[j] = in && e < d ? *reinterpret_cast<const uint32_t*>(
                                         s + static_cast<int64_t>(e) * n + n0 + t)
                                   : 0u;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = e0 + j * kRows;
                if (e >= d) break;
                float* to = tile + tile_row(e, quarter) * (TT + 1) + t;
                to[0] = bf16_to_f32(v[j] & 0xffffu);
                to[1] = __uint_as_float(v[j] & 0xffff0000u);
            }
        }
        return;
    }
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
            if (e < d) tile[tile_row(e, quarter) * (TT + 1) + t] = v[j];
        }
    }
}

template <class T, int TT>
__device__ __forceinline__ void tile_store(void* dst, int64_t n, int d, int64_t n0, bool pairs,
                                           const float* tile) {
    const int quarter = tile_quarter(d);
    if (T::kBytes == 2 && pairs) {
        constexpr int kCols = TT / 2, kRows = kTileThreads / kCols;
        const int t = 2 * (threadIdx.x % kCols);
        if (n0 + t >= n) return;
        uint16_t* to = static_cast<uint16_t*>(dst);
        for (int e = threadIdx.x / kCols; e < d; e += kRows) {
            const float* x = tile + tile_row(e, quarter) * (TT + 1) + t;
            *reinterpret_cast<uint32_t*>(to + static_cast<int64_t>(e) * n + n0 + t) =
                f32_to_bf16(x[0]) | (static_cast<uint32_t>(f32_to_bf16(x[1])) << 16);
        }
        return;
    }
    const int t = threadIdx.x % TT;
    if (n0 + t >= n) return;
    for (int e = threadIdx.x / TT; e < d; e += kTileThreads / TT)
        T::store(dst, static_cast<int64_t>(e) * n + n0 + t,
                 tile[tile_row(e, quarter) * (TT + 1) + t]);
}

// Tokens of a tile: 32 (128 bytes of a float32 feature) where it takes at most
// `lds` bytes and the workgroups still fill the card, else 16.
inline int tile_tokens(int64_t n, int64_t d, int64_t lds) {
    return 4 * tile_quarter(d) * 33 * 4 <= lds && n >= 32 * kTileMinGroups ? 32 : 16;
}

inline bool tile_pairs(const slk_norm* a, std::initializer_list<const void*> cols) {
    if (a->dtype != SLK_BF16 || a->n % 2 != 0) return false;
    for (const void* p : cols)
        if (p != nullptr && !aligned_to(p, 4)) return false;
    return true;
}

template <int EPL, int TT, bool VEC>
__device__ __forceinline__ void tile_row_load(const float* tile, int t, int d, int l,
                                              float (&v)[EPL]) {
    const int quarter = tile_quarter(d);
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = RowLay<EPL, 1, VEC>::at(q, l);
        v[q] = e < d ? tile[tile_row(e, quarter) * (TT + 1) + t] : 0.0f;
    }
}

template <int EPL, int TT, bool VEC>
__device__ __forceinline__ void tile_row_store(float* tile, int t, int d, int l,
                                               const float (&v)[EPL]) {
    const int quarter = tile_quarter(d);
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = RowLay<EPL, 1, VEC>::at(q, l);
        if (e < d) tile[tile_row(e, quarter) * (TT + 1) + t] = v[q];
    }
}

// A token-major row fetched ahead (AHEAD), or loaded when asked for.
template <class T, int EPL, bool VEC, bool AHEAD>
struct Ahead {
    RawRow<T, EPL, 1> raw;
    __device__ __forceinline__ void fetch(const void* p, int64_t off, int d, int l) {
        if constexpr (VEC && AHEAD) raw.load(p, off, d, l);
    }
    __device__ __forceinline__ void get(const void* p, int64_t off, int d, int l,
                                        float (&v)[EPL]) const {
        if constexpr (VEC && AHEAD) raw.get(v);
        else row_load<T, EPL, 1, VEC>(p, off, d, l, v);
    }
};

}  // namespace slk
