// Attention of a few new tokens over long key and value arrays, read where they
// lie (slk_attention_forward with few queries and no backward to follow).
//
// The matrix cores have little to multiply here: a key or value is used by the
// handful of rows (new tokens times the query heads of its group), and reading it
// is the work. A key's row lies over DP/8 lanes, eight elements each, so a wave
// reads 64 / (DP/8) keys with one or two 16-byte loads a lane, four such groups in
// flight; a score is eight fused multiply-adds and a sum over those lanes (DPP).
// Every group of lanes keeps its own running maximum, sum and weighted values of
// up to four rows (eight took registers that left one wave a SIMD: slower than
// reading the keys twice, the second time from the L2); they are joined once at the
// end, over lanes, waves and, where the keys are split over workgroups to fill the
// card, by the join kernel. 16 sequences of 7236 keys in the mean, 8 heads of 128,
// bfloat16, 474 MB: 105 us, 4.5 TB/s (and 5 for the join); one of 106147 keys, 12 heads of
// 64, float32, a bias, 652 MB: 126 us, 5.2 TB/s. Rows beyond four read the keys again: 4 x
// 16384 keys, 8 heads of 128, bfloat16, 57 us at a large copy's rate: 65 us with 4 rows a key
// head, 104 with 8, 183 with 16.
#include "attention_decode.hpp"

namespace slk {

namespace {

constexpr int kDecodeWaves = 4, kInFlight = 4;

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(__float_as_uint(x)), CTRL, 0xf, 0xf, true)));
}

// Sum over aligned groups of L lanes, in every lane.
template <int L>
__device__ __forceinline__ float lane_sum(float x) {
    if constexpr (L >= 16) x += dpp<0x140>(x);  // row mirror
    if constexpr (L >= 8) x += dpp<0x141>(x);   // half-row mirror
    x += dpp<0x4e>(x);                          // lanes 2, 3, 0, 1 of four
    x += dpp<0xb1>(x);                          // lanes 1, 0, 3, 2
    return x;
}

// Eight consecutive features of a row as they are loaded. The fast form: dim a
// multiple of 8, rows of consecutive features, 16-byte aligned; lanes past dim read
// the row's first features (their part of the query is zero).
template <class IO>
struct Raw;
template <>
struct Raw<F32> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const AttnIo& x, int64_t at, int f, int dim, bool vec) {
        if (vec) {
            const f32x4* p = reinterpret_cast<const f32x4*>(x.p + 4 * (at + (f < dim ? f : 0)));
            a = p[0];
            b = p[1];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[j] = f + j < dim ? F32::load(x.p, at + (f + j) * x.sd) : 0.0f;
                b[j] = f + 4 + j < dim ? F32::load(x.p, at + (f + 4 + j) * x.sd) : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    }
};
template <>
struct Raw<BF16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const AttnIo& x, int64_t at, int f, int dim, bool vec) {
        if (vec) {
            const uint4 a = *reinterpret_cast<const uint4*>(x.p + 2 * (at + (f < dim ? f : 0)));
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(x.p);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int g = f + 2 * j;
                const uint32_t lo = g < dim ? p[at + g * x.sd] : 0;
                const uint32_t hi = g + 1 < dim ? p[at + (g + 1) * x.sd] : 0;
                w[j] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
};

template <class IO, int DB, int R, bool BIAS>
__global__ __launch_bounds__(64 * kDecodeWaves) void attn_decode_kernel(const AttnDecode a) {
    constexpr int L = 4 * DB, KP = kWave / L, DP = 32 * DB;
    constexpr int kStep = KP * kInFlight;  // keys of a wave's pass
    __shared__ float join_ml[kDecodeWaves][R][2];
    __shared__ float join_o[kDecodeWaves][R][DP];
    extern __shared__ float bias_rows[];

    const AttnArgs& g = a.g;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rep = g.heads / g.kv_heads;
    uint32_t u = blockIdx.x;
    const int kvh = u % g.kv_heads;
    u /= g.kv_heads;
    const int chunk = u % a.chunks;
    u /= a.chunks;
    const int split = u % g.splits;
    const int sid = u / g.splits;
    AttnSeq seq = attn_seq(g.plan, sid);
    if (a.k_lengths != nullptr) seq.nk = max(0, min(a.k_lengths[sid], seq.nk));
    const int n_rows = rep * seq.eq, r0 = chunk * R;  // row r: query r / rep, head r % rep
    if (r0 >= n_rows) return;
    const int shift = seq.nk - seq.nq;

    const int per = ((seq.nk + g.splits - 1) / g.splits + kStep - 1) / kStep * kStep;
    const int k_lo = static_cast<int>(min(static_cast<int64_t>(split) * per,
                                          static_cast<int64_t>(seq.nk)));
    const int k_hi = static_cast<int>(min(static_cast<int64_t>(k_lo) + per,
                                          static_cast<int64_t>(seq.nk)));
    const int md = BIAS ? g.bias.max_distance : 0, width = 2 * md + 1;
    if constexpr (BIAS) {
        for (int r = 0; r < R && r0 + r < n_rows; ++r)
            for (int i = threadIdx.x; i < width; i += 64 * kDecodeWaves)
                bias_rows[r * width + i] =
                    attn_bias_of(g.bias, g.heads, kvh * rep + (r0 + r) % rep, i - md);
        __syncthreads();
    }

    const int f = 8 * (lane % L), slot = lane / L;
    float q[R][8], o[R][8], m[R], l[R];
    int at[R], lim[R];  // a row's position among the keys, and the last key that it sees
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = min(r0 + r, n_rows - 1), t = i / rep, h = kvh * rep + i % rep;
        Raw<IO> raw;
        raw.load(a.q, sid * a.q.sb + (seq.q0 + min(t, max(seq.nq - 1, 0))) * a.q.sr + h * a.q.sh,
                 f, g.dim, false);
        raw.get(q[r]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q[r][j] *= g.scale2;
            o[r][j] = 0.0f;
        }
        m[r] = -INFINITY;
        l[r] = 0.0f;
        at[r] = t + shift;
        lim[r] = t >= seq.nq ? -1 : g.causal ? min(seq.nk - 1, at[r]) : seq.nk - 1;
    }
    int lim_lo = lim[0];
#pragma unroll
    for (int r = 1; r < R; ++r) lim_lo = min(lim_lo, lim[r]);

    const int64_t kb = sid * a.k.sb + static_cast<int64_t>(seq.k0) * a.k.sr + kvh * a.k.sh;
    const int64_t vb = sid * a.v.sb + static_cast<int64_t>(seq.k0) * a.v.sr + kvh * a.v.sh;
    // The next pass's keys are asked for when this one's are in the scores, its
    // values when this one's are added: one or the other is always on its way.
    Raw<IO> rk[kInFlight], rv[kInFlight];
    auto load = [&](Raw<IO>(&to)[kInFlight], const AttnIo& x, int64_t base, int key0)
        __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const int64_t key = min(key0 + i * KP + slot, k_hi - 1);
            to[i].load(x, base + key * x.sr, f, g.dim, a.vec);
        }
    };
    constexpr int kNext = kDecodeWaves * kStep;
    if (k_lo + wv * kStep < k_hi) {
        load(rk, a.k, kb, k_lo + wv * kStep);
        load(rv, a.v, vb, k_lo + wv * kStep);
    }
    for (int key0 = k_lo + wv * kStep; key0 < k_hi; key0 += kNext) {
        const bool masked = key0 + kStep > k_hi || key0 + kStep - 1 > lim_lo;
        float s[R][kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            float x[8];
            rk[i].get(x);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float z = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) z = __builtin_fmaf(x[j], q[r][j], z);
                s[r][i] = lane_sum<L>(z);
                if constexpr (BIAS)
                    s[r][i] += bias_rows[r * width + md +
                                         attn_clamp(at[r] - (key0 + i * KP + slot), md)];
            }
        }
        if (key0 + kNext < k_hi) load(rk, a.k, kb, key0 + kNext);
        uint32_t see = ~0u;  // bit 4 r + i
        if (masked) {
            see = 0;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < kInFlight; ++i) {
                    const int key = key0 + i * KP + slot;
                    const bool in = key < k_hi && key <= lim[r];
                    s[r][i] = in ? s[r][i] : -INFINITY;
                    see |= (in ? 1u : 0u) << (kInFlight * r + i);
                }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = s[r][0];
#pragma unroll
            for (int i = 1; i < kInFlight; ++i) top = fmaxf(top, s[r][i]);
            if (top > m[r]) {
                const float scale = attn_exp2(m[r] - top);
                m[r] = top;
                l[r] *= scale;
#pragma unroll
                for (int j = 0; j < 8; ++j) o[r][j] *= scale;
            }
            const float ref = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) {
                s[r][i] = attn_exp2(s[r][i] - ref);
                l[r] += s[r][i];
            }
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            float y[8];
            rv[i].get(y);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (masked) {  // a value that is not seen may be anything
                    const bool in = (see >> (kInFlight * r + i)) & 1;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        o[r][j] = in ? __builtin_fmaf(s[r][i], y[j], o[r][j]) : o[r][j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        o[r][j] = __builtin_fmaf(s[r][i], y[j], o[r][j]);
                }
            }
        }
        if (key0 + kNext < k_hi) load(rv, a.v, vb, key0 + kNext);
    }

    // over the wave's groups of lanes, then over the waves
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int x = L; x < kWave; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float scale = m[r] == -INFINITY ? (l[r] == 0.0f ? 0.0f : l[r]) : attn_exp2(m[r] - top);
        l[r] *= scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[r][j] = l[r] == 0.0f && scale == 0.0f ? 0.0f : o[r][j] * scale;
#pragma unroll
        for (int x = L; x < kWave; x <<= 1) {
            l[r] += __shfl_xor(l[r], x);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[r][j] += __shfl_xor(o[r][j], x);
        }
        if (lane == 0) {
            join_ml[wv][r][0] = top;
            join_ml[wv][r][1] = l[r];
        }
        if (slot == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) join_o[wv][r][f + j] = o[r][j];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * DP; i += 64 * kDecodeWaves) {
        const int r = i / DP, e = i % DP;
        if (r0 + r >= n_rows) break;
        float top = -INFINITY;
        for (int w = 0; w < kDecodeWaves; ++w) top = fmaxf(top, join_ml[w][r][0]);
        float sum = 0.0f, x = 0.0f;
        for (int w = 0; w < kDecodeWaves; ++w) {
            const float part = join_ml[w][r][1];
            if (part == 0.0f) continue;
            const float scale = attn_exp2(join_ml[w][r][0] - top);
            sum = __builtin_fmaf(part, scale, sum);
            x = __builtin_fmaf(join_o[w][r][e], scale, x);
        }
        const int t = (r0 + r) / rep, head = kvh * rep + (r0 + r) % rep;
        if (g.splits > 1) {
            if (t >= seq.nq) continue;
            const int64_t row =
                (static_cast<int64_t>(split) * g.heads + head) * g.part_rows + seq.pq + t;
            if (e == 0) {
                g.part_ml[2 * row] = top;
                g.part_ml[2 * row + 1] = sum;
            }
            g.part[row * DP + e] = x;
        } else if (e < g.dim) {
            const int64_t to = sid * g.out.sb + (seq.q0 + t) * g.out.sr + head * g.out.sh +
                               e * g.out.sd;
            IO::store(g.out.p, to, t < seq.nq && sum != 0.0f ? x / sum : 0.0f);
        }
    }
}

template <class IO, int DB, int R>
int launch(const AttnDecode& a, int64_t groups, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(groups)), wg(64 * kDecodeWaves);
    if (a.g.bias.table != nullptr) {
        const size_t lds = R * (2 * a.g.bias.max_distance + 1) * sizeof(float);
        hipLaunchKernelGGL((attn_decode_kernel<IO, DB, R, true>), grid, wg, lds, st, a);
    } else {
        hipLaunchKernelGGL((attn_decode_kernel<IO, DB, R, false>), grid, wg, 0, st, a);
    }
    return check_launch("attention_forward: few queries");
}

template <class IO, int DB>
int launch_rows(const AttnDecode& a, int rows, int64_t groups, hipStream_t st) {
    if (rows == 1) return launch<IO, DB, 1>(a, groups, st);
    if (rows == 2) return launch<IO, DB, 2>(a, groups, st);
    return launch<IO, DB, 4>(a, groups, st);
}

template <class IO>
int launch_dim(const AttnDecode& a, int db, int rows, int64_t groups, hipStream_t st) {
    if (db == 1) return launch_rows<IO, 1>(a, rows, groups, st);
    if (db == 2) return launch_rows<IO, 2>(a, rows, groups, st);
    return launch_rows<IO, 4>(a, rows, groups, st);
}

}  // namespace

int attn_launch_decode(const AttnDecode& a, int db, int rows, hipStream_t st) {
    const int64_t groups = a.g.plan.batch * a.g.splits * a.chunks * a.g.kv_heads;
    if (groups > max_groups(64 * kDecodeWaves))
        return fail(SLK_EINVAL, "attention_forward: too many sequences");
    const int rc = a.g.dtype == SLK_F32 ? launch_dim<F32>(a, db, rows, groups, st)
                                        : launch_dim<BF16>(a, db, rows, groups, st);
    if (rc != SLK_OK || a.g.splits == 1) return rc;
    return attn_launch_join(a.g, db, st);
}

}  // namespace slk
