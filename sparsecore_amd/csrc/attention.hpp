// Attention between projections, forward and backward (slk_attention_*): what
// its kernels share.
//
//   S = scale·Q·K^T (+ bias of the distance),  P = softmax of S over the keys a
//   query sees,  O = P·V;
//   dV = P^T·dO,  dP = dO·V^T,  dS = P∘(dP - rowsum(dO∘O)),
//   dQ = scale·dS·K,  dK = scale·dS^T·Q,  dbias = dS summed over a bucket's pairs.
//
// Scores are in units of log 2 (scale and bias times log2 e), so that the
// exponentials are the hardware's.
//
// Operands. The matrix cores take 16-bit elements. bfloat16 tensors whose rows
// are 16-byte pieces are read where they lie; everything else (float32, other
// strides, a head size between 32, 64 and 128) is packed first, head by head, a
// sequence's rows from a multiple of 64 on and zero behind its last. A float32
// x is packed as two float16 parts of x·2^(14 - e), e the exponent of the
// largest of its 32 rows of one head: hi + lo keep 22 bits of x down to 2^-39 of
// that largest. Products take hi·hi + hi·lo + lo·hi, about float32's own
// rounding at a third of the float16 rate; the powers of two are uniform over a
// block of 32 x 32 and cost nothing there: they go into factors that each
// element is multiplied by anyway.
#pragma once

#include "mma_tile.hpp"

namespace slk {

constexpr int kAttnRows = 64;     // rows of a staged tile, and what packed sequences are padded to
constexpr int kAttnThreads = 256;
constexpr int kAttnUnit = 14;     // a packed float32 tile's largest element is in 2^[14, 15)
constexpr float kLog2e = 1.44269504088896340736f;

// One sequence: rows [q0, q0 + nq) of its batch entry are queries, nq of eq rows
// that the call writes; keys likewise. pq, pk: first padded row.
struct AttnSeq {
    int32_t q0, nq, eq, k0, nk, ek, pq, pk;
};

// Sequences and the order of their tiles. Uniform (seqs NULL): batch entries of
// t and s rows. Else seqs, and lists of (sequence, tile), most work first.
struct AttnPlan {
    const AttnSeq* seqs;
    const int2* list;
    const int32_t* count;
    int64_t batch, t, s;
    int64_t pad_t, pad_s;
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnPlan& p, int s) {
    if (p.seqs != nullptr) return p.seqs[s];
    AttnSeq q;
    q.q0 = q.k0 = 0;
    q.nq = q.eq = static_cast<int32_t>(p.t);
    q.nk = q.ek = static_cast<int32_t>(p.s);
    q.pq = static_cast<int32_t>(s * p.pad_t);
    q.pk = static_cast<int32_t>(s * p.pad_s);
    return q;
}

// Entry e of the tile order: sequence and tile. first_long: tile 0 has the most
// work (keys of a causal mask), else the last one.
__device__ __forceinline__ bool attn_entry(const AttnPlan& p, int64_t e, int64_t tiles,
                                           bool first_long, int& seq, int& tile) {
    if (p.seqs != nullptr) {
        if (e >= *p.count) return false;
        const int2 x = p.list[e];
        seq = __builtin_amdgcn_readfirstlane(x.x);
        tile = __builtin_amdgcn_readfirstlane(x.y);
        return true;
    }
    const int64_t rank = e / p.batch;
    seq = static_cast<int>(e - rank * p.batch);
    tile = static_cast<int>(first_long ? rank : tiles - 1 - rank);
    return rank < tiles;
}

// A 16-bit operand as the kernels read it; strides in bytes. Packed: padded rows
// of planes hi, lo; else the caller's tensor.
struct AttnOp {
    const char* p;
    int64_t sb, sr, sh;
    int32_t plane;         // bytes from the high to the low part
    int32_t packed;
    const int32_t* exps;   // [head][padded rows / 32]; NULL: bfloat16
    int64_t exps_sh;
    __device__ __forceinline__ const char* rows(int seq, int first, int padded, int head) const {
        return packed ? p + head * sh + padded * sr : p + seq * sb + head * sh + first * sr;
    }
};

// A caller's tensor, strides in elements.
struct AttnIo {
    char* p;
    int64_t sb, sr, sh, sd;
};

struct AttnBias {
    const void* table;  // buckets x heads; NULL: none
    int32_t dtype, buckets, max_distance, one_sided;
    uint16_t starts[SLK_ATTN_MAX_BUCKETS];  // first distance of each bucket of one side
};

struct AttnArgs {
    AttnPlan plan;
    AttnOp q, k, v, dout;
    AttnIo out, dq, dk, dv;
    float* lse;            // [head][padded row]: log2 of the sum; +inf: no key seen, or no query
    float* delta;          // [head][padded row]: rowsum(dO∘O)
    int32_t* dexps;        // [head][padded rows / 32]: exponent of the largest |delta|
    int64_t lse_sh;
    AttnBias bias;
    float* dbias_part;     // [head][padded rows / 64][2·max_distance + 1]
    int64_t dbias_slots;
    float* part;           // split keys: [split][head][padded row][DP] of O, then of m, l
    float* part_ml;
    int64_t part_rows;
    int32_t splits;
    int32_t heads, kv_heads, dim, dtype, causal;
    int64_t tiles;         // of the uniform plan
    float scale2, scale;   // scale·log2 e, scale
};

// A staged plane: 64 rows of DP 16-bit elements, 16-byte pieces permuted so that
// the 16 lanes of an LDS pass meet all banks once, both where they read one piece
// of 16 consecutive rows (along) and where they read 64 bytes of each of four
// rows (across, the transposing read).
template <int DB>
struct AttnTile {
    static constexpr int DP = 32 * DB, kPieces = DP / 8, kRowBytes = 2 * DP;
    static constexpr int kPlane = kAttnRows * kRowBytes;
    static constexpr int kChunks = kPlane / 1024;  // direct loads of a plane
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (DB == 4) return ((row & 3) << 2) | ((row >> 2) & 3);
        else if constexpr (DB == 2) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else return (row >> 2) & 3;
    }
};

template <bool SPLIT>
using AttnFrag = std::conditional_t<SPLIT, f16x8, b16x8>;

template <bool SPLIT>
__device__ __forceinline__ f32x16 attn_mfma(AttnFrag<SPLIT> a, AttnFrag<SPLIT> b, f32x16 c) {
    if constexpr (SPLIT) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Operand fragments with their parts, and their product.
template <bool SPLIT>
struct AttnPair {
    AttnFrag<SPLIT> f[SPLIT ? 2 : 1];
};
template <bool SPLIT>
__device__ __forceinline__ f32x16 attn_dot(const AttnPair<SPLIT>& a, const AttnPair<SPLIT>& b,
                                           f32x16 c) {
    if constexpr (SPLIT) {
        c = attn_mfma<true>(a.f[1], b.f[0], c);
        c = attn_mfma<true>(a.f[0], b.f[1], c);
        return attn_mfma<true>(a.f[0], b.f[0], c);
    } else {
        return attn_mfma<false>(a.f[0], b.f[0], c);
    }
}

// The direct loads of one operand's tiles of 64 rows: wave wv takes chunks
// wv, wv + 4, ... of each plane. Rows past the last one (n live rows) read it again.
template <bool SPLIT, int DB, int WAVES = 4>
struct AttnLoads {
    using T = AttnTile<DB>;
    static constexpr int kPer = (T::kChunks + WAVES - 1) / WAVES;
    const char* base;
    int64_t sr;
    int32_t plane, last;
    int row[kPer], piece[kPer];
    __device__ __forceinline__ AttnLoads(const AttnOp& op, const char* b, int n, int wv, int lane)
        : base(b), sr(op.sr), plane(op.plane), last(n - 1) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = (wv + WAVES * i) * 64 + lane;
            row[i] = at / T::kPieces;
            piece[i] = 16 * ((at % T::kPieces) ^ T::swz(row[i]));
        }
    }
    __device__ __forceinline__ void issue(unsigned char* to, int r0, int wv,
                                          int64_t more = 0) const {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass emits no stub of a kernel that calls this
        const uint64_t at = reinterpret_cast<uint64_t>(base + r0 * sr + more);
        const int left = last - r0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (T::kChunks % WAVES != 0 && wv + WAVES * i >= T::kChunks) break;
            const uint32_t off =
                static_cast<uint32_t>(row[i] < left ? row[i] : left) * static_cast<uint32_t>(sr) +
                piece[i];
#pragma unroll
            for (int p = 0; p < (SPLIT ? 2 : 1); ++p) {
                const uint64_t from = at + (p ? plane : 0);
                const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(from));
                const uint32_t hi =
                    __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(from >> 32));
                const char* src =
                    reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
                uint32_t o = off;
                asm("" : "+v"(o));
                __builtin_amdgcn_global_load_lds(
                    src + o, to + p * T::kPlane + 1024 * (wv + WAVES * i), 16, 0, 0);
            }
        }
#endif
    }
};

// Reads of a staged operand by one lane. along: row l % 32 of a block of 32 rows,
// features 16 ks + 8 (l / 32) ...: the rows are the product's. across: feature
// 32 fb + l % 32, rows 16 s + 8 (j / 4) + 4 (l / 32) + j % 4 for j = 0..7 of a
// block of 32: the rows are summed over, in the order in which a lane holds them
// in a product's result (register 8 s + j), so that a result goes into the next
// product from the registers that it is in.
template <bool SPLIT, int DB>
struct AttnReads {
    using T = AttnTile<DB>;
    int lane;
    __device__ __forceinline__ explicit AttnReads(int l) : lane(l) {}
    __device__ __forceinline__ AttnPair<SPLIT> along(const unsigned char* buf, int b,
                                                     int ks) const {
        const int row = 32 * b + (lane & 31), piece = 2 * ks + (lane >> 5);
        AttnPair<SPLIT> r;
#pragma unroll
        for (int p = 0; p < (SPLIT ? 2 : 1); ++p)
            r.f[p] = *reinterpret_cast<const AttnFrag<SPLIT>*>(
                buf + p * T::kPlane + row * T::kRowBytes + 16 * (piece ^ T::swz(row)));
        return r;
    }
    __device__ __forceinline__ AttnPair<SPLIT> across(const unsigned char* buf, int b, int s,
                                                      int fb) const {
        const int i = lane & 15;
        const int piece = 4 * fb + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1);
        AttnPair<SPLIT> r;
#pragma unroll
        for (int p = 0; p < (SPLIT ? 2 : 1); ++p) {
            i16x4 x[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = 32 * b + 16 * s + 8 * u + 4 * (lane >> 5) + (i >> 2);
                x[u] = read_turned(buf + p * T::kPlane + row * T::kRowBytes +
                                   16 * (piece ^ T::swz(row)) + 8 * (i & 1));
            }
            r.f[p] = __builtin_bit_cast(
                AttnFrag<SPLIT>, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return r;
    }
};

// Eight results of a lane as an operand: rounded to bfloat16 (relative 2^-8, of
// weights and of their gradients, as the tensors themselves are), or in two
// float16 parts (22 bits).
template <bool SPLIT>
__device__ __forceinline__ AttnPair<SPLIT> attn_operand(const float* x) {
    AttnPair<SPLIT> r;
    if constexpr (SPLIT) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const _Float16 h = static_cast<_Float16>(x[j]);
            r.f[0][j] = h;
            r.f[1][j] = static_cast<_Float16>(x[j] - static_cast<float>(h));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r.f[0][j] = static_cast<__bf16>(x[j]);
    }
    return r;
}

// Bits of a fragment that are not finite, as 1.0 where they are and 0 elsewhere,
// and the fragment with zeros there.
template <bool SPLIT>
__device__ __forceinline__ bool attn_split_finite(AttnPair<SPLIT>& a, AttnFrag<SPLIT>& bad) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    constexpr uint16_t kExp = SPLIT ? 0x7c00 : 0x7f80, kOne = SPLIT ? 0x3c00 : 0x3f80;
    u16x8 x[SPLIT ? 2 : 1], one;
#pragma unroll
    for (int p = 0; p < (SPLIT ? 2 : 1); ++p) x[p] = __builtin_bit_cast(u16x8, a.f[p]);
    bool any = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bool b = (x[0][j] & kExp) == kExp;
        if constexpr (SPLIT) b = b || (x[1][j] & kExp) == kExp;
        any = any || b;
        one[j] = b ? kOne : 0;
#pragma unroll
        for (int p = 0; p < (SPLIT ? 2 : 1); ++p) x[p][j] = b ? 0 : x[p][j];
    }
#pragma unroll
    for (int p = 0; p < (SPLIT ? 2 : 1); ++p) a.f[p] = __builtin_bit_cast(AttnFrag<SPLIT>, x[p]);
    bad = __builtin_bit_cast(AttnFrag<SPLIT>, one);
    return any;
}

template <bool SPLIT>
__device__ __forceinline__ bool attn_any_bad(const AttnPair<SPLIT>& a) {
    AttnPair<SPLIT> c = a;
    AttnFrag<SPLIT> bad;
    return attn_split_finite<SPLIT>(c, bad);
}

// acc[fb] += X^T·W over one block of 32 staged rows X, where W (a lane's 16
// results, zero where the pair is masked) is given as its operands and `seen` has
// a bit for each of the 16. A zero weight must also silence a row that is not
// finite: 0 · inf is NaN. So where a block has masked pairs and X a value that
// is not finite, the product takes zeros there, and the results whose sum has
// such a term become NaN.
template <bool SPLIT, int DB, int NB>
__device__ __forceinline__ void attn_accumulate(const AttnReads<SPLIT, DB>& rd,
                                                const unsigned char* buf, int b,
                                                const AttnPair<SPLIT> (&w)[NB][2],
                                                f32x16 (&acc)[DB][NB], bool masked,
                                                const uint32_t (&seen)[NB]) {
#pragma unroll
    for (int fb = 0; fb < DB; ++fb) {
        AttnPair<SPLIT> x[2] = {rd.across(buf, b, 0, fb), rd.across(buf, b, 1, fb)};
        if (masked && __builtin_amdgcn_ballot_w64(attn_any_bad<SPLIT>(x[0]) ||
                                                  attn_any_bad<SPLIT>(x[1])) != 0) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                f32x16 cnt;
#pragma unroll
                for (int r = 0; r < 16; ++r) cnt[r] = 0.0f;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    AttnPair<SPLIT> c = x[s];
                    AttnFrag<SPLIT> bad, on;
                    attn_split_finite<SPLIT>(c, bad);
                    using E = std::conditional_t<SPLIT, _Float16, __bf16>;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        on[j] = static_cast<E>(((seen[n] >> (8 * s + j)) & 1) ? 1.0f : 0.0f);
                    cnt = attn_mfma<SPLIT>(bad, on, cnt);
                    acc[fb][n] = attn_dot<SPLIT>(c, w[n][s], acc[fb][n]);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[fb][n][r] = cnt[r] > 0.0f ? __builtin_nanf("") : acc[fb][n][r];
            }
        } else {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    acc[fb][n] = attn_dot<SPLIT>(x[s], w[n][s], acc[fb][n]);
        }
    }
}

// Row (in a block of 32) that register r of a result belongs to.
__device__ __forceinline__ int attn_row(int r, int lane) {
    return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^e for any e; 0 below the smallest.
__device__ __forceinline__ float attn_pow2(int e) { return ldexpf(1.0f, e); }

__device__ __forceinline__ int attn_exp(const AttnOp& op, int head, int padded_row) {
    return __builtin_amdgcn_readfirstlane(op.exps[head * op.exps_sh + (padded_row >> 5)]);
}

// The bias of each distance query - key in [-max_distance, max_distance], times
// log2 e, from the buckets' table into LDS (all threads; a barrier follows).
__device__ __forceinline__ void attn_bias_row(const AttnBias& b, int heads, int head, float* row) {
    const int one = b.one_sided ? b.buckets : b.buckets / 2;
    for (int i = threadIdx.x; i <= 2 * b.max_distance; i += blockDim.x) {
        const int away = i - b.max_distance, n = away < 0 ? -away : away;
        int lo = 0, hi = one;  // the last bucket that starts at or before n
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (b.starts[mid] <= n) lo = mid;
            else hi = mid;
        }
        const int bucket = lo + (!b.one_sided && away < 0 ? one : 0);
        const int64_t at = static_cast<int64_t>(bucket) * heads + head;
        const float x = b.dtype == SLK_F32 ? static_cast<const float*>(b.table)[at]
                                           : bf16_to_f32(static_cast<const uint16_t*>(b.table)[at]);
        row[i] = x * kLog2e;
    }
}

__device__ __forceinline__ int attn_clamp(int x, int m) { return x < -m ? -m : x > m ? m : x; }

// Sixteen results of a lane, features 32 fb + attn_row(r) of one row, to a
// caller's tensor at `at` (elements). Four consecutive features in one store
// where they are consecutive in memory and aligned.
template <class IO>
__device__ __forceinline__ void attn_store(const AttnIo& t, int64_t at, int fb, int lane, int dim,
                                           bool vec, const f32x16& x, float factor) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
        const int f = 32 * fb + 8 * r4 + 4 * (lane >> 5);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[4 * r4 + j] * factor;
        if (vec) {
            if (f < dim) IO::store4(t.p, at + f, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (f + j < dim) IO::store(t.p, at + (f + j) * t.sd, v[j]);
        }
    }
}

int attn_launch_forward(const AttnArgs& g, bool split, int db, int64_t entries, hipStream_t st);
int attn_launch_backward(const AttnArgs& g, bool split, int db, const AttnPlan& kplan,
                         int64_t q_entries, int64_t k_entries, bool want_q, bool want_kv,
                         int64_t k_tiles, hipStream_t st);
// joins the parts of split keys
int attn_launch_join(const AttnArgs& g, int db, hipStream_t st);
int attn_launch_dbias(const AttnArgs& g, void* dbias, hipStream_t st);

}  // namespace slk
