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
// Operands. The matrix cores take float16 here, of both types. Every operand is
// packed first, head by head, a sequence's rows from a multiple of 64 on and zero
// behind its last: whatever its strides and head size are, the kernels then copy
// tiles of 64 rows into LDS as they lie. A tile's elements are multiplied by
// 2^(14 - e), e the exponent of its largest one. A bfloat16 element (8 bits) is
// then exact down to 2^-31 of the tile's largest. A float32 one becomes two
// parts, hi + lo, which keep 22 bits down to 2^-39; products take hi·hi + hi·lo +
// lo·hi, about float32's own rounding at a third of the float16 rate. The powers
// of two are uniform over a block and cost nothing: they go into factors that
// each element is multiplied by anyway.
// A tile with a row whose largest element is 2^-kAttnSpread or less of the tile's is
// uneven: each of its rows has an exponent of its own, so that no row, least of all one
// that others do not see, takes bits off another: an element is then off by 2^-22 of
// itself or 2^-25 of its row's largest (bfloat16: exact down to 2^-17 of that). A
// workgroup that meets such a tile takes a second form of its loop, which applies
// exponents row by row. 16384 tokens, 32 heads over 8 of 128, bfloat16, all tiles uneven:
// forward 4.0 ms in place of 2.4, backward 12.6 in place of 8.3; the look at the tiles'
// flags costs 1 us a kernel. Values that are not finite are packed as
// zeros (masked, they would make 0 · inf of a zero weight) and their rows noted:
// the forward makes NaN of what sees them, log-sums included, from which the
// backward's weights are NaN in their turn. bfloat16 products would save the packing
// (a fiftieth of a long sequence's time), but weights and their gradients would
// be rounded to 8 bits on the way: errors of the gradients of 1.7 times the
// rounding of the result alone.
#pragma once

#include "mma_tile.hpp"

namespace slk {

constexpr int kAttnRows = 64;     // rows of a staged tile, and what packed sequences are padded to
constexpr int kAttnTileRows = 128; // rows of a workgroup of the tiled kernels
constexpr int kAttnThreads = 256;
constexpr int kAttnMaxSplits = 128;  // parts of the keys
constexpr int kAttnUnit = 14;     // a packed tile's largest element is in 2^[14, 15)
constexpr int kAttnSpread = 14;   // of the exponents of an even tile's rows
constexpr int kUnset = -100000;   // the exponent of a row's unit before it has seen anything
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
    const int32_t *q_map, *k_map;  // the sequence of each tile of 64 padded rows
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

// Sequence and row in it of a padded row of queries or keys; rows past the last
// sequence's have none.
struct AttnRow {
    int sid, row;
    AttnSeq seq;
    bool any;
};
__device__ __forceinline__ AttnRow attn_row_of(const AttnPlan& p, bool keys, int64_t padded) {
    AttnRow r;
    if (p.seqs == nullptr) {
        const int64_t pad = keys ? p.pad_s : p.pad_t;
        r.sid = static_cast<int>(padded / pad);
        r.any = r.sid < p.batch;
        r.seq = attn_seq(p, r.sid);
        r.row = static_cast<int>(padded - r.sid * pad);
        return r;
    }
    r.sid = (keys ? p.k_map : p.q_map)[padded >> 6];
    r.any = r.sid >= 0;
    if (!r.any) return r;
    r.seq = p.seqs[r.sid];
    r.row = static_cast<int>(padded - (keys ? r.seq.pk : r.seq.pq));
    return r;
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

// A packed operand: tiles of 64 rows, each as it lies in LDS (AttnTile), planes of
// high and low parts one behind the other.
struct AttnOp {
    const char* p;
    int64_t sh;            // bytes of a head
    // [head][tile]: 4·exponent, + 2 where the tile is uneven, + 1 where a value is not finite
    const int32_t* exps;
    const uint64_t* bad;   // [head][tile]: a bit for each row with such values
    const int8_t* rows;    // [head][padded row]: the exponent that the row is packed with
    int64_t exps_sh;       // tiles of a head
    __device__ __forceinline__ const int8_t* row(int head, int64_t padded) const {
        return rows + head * exps_sh * kAttnRows + padded;
    }
};

// A caller's tensor, strides in elements.
struct AttnIo {
    char* p;
    int64_t sb, sr, sh, sd;
};

struct AttnBias {
    const void* table;  // buckets x heads; NULL: none
    float* rows;        // [head][2·max_distance + 1]: the bias of each distance, times log2 e
    int32_t dtype, buckets, max_distance, one_sided;
    uint16_t starts[SLK_ATTN_MAX_BUCKETS];  // first distance of each bucket of one side
};

struct AttnArgs {
    AttnPlan plan;
    AttnOp q, k, v, dout;
    AttnIo out, dq, dk, dv;
    float* lse;            // [head][padded row]: log2 of the sum; +inf: no key seen, or no query;
                           // NaN: a value that is not finite is seen
    float* inv;            // with biases, lse is the row's maximum and inv 1 / the sum below it:
                           // a bias of the type's lowest value would swallow the logarithm
    float* delta;          // [head][padded row]: rowsum(dO∘O)
    int32_t* dexps;        // [head][padded rows / 64]: exponent of the largest |delta|
    int64_t lse_sh;
    char* o_rest;          // what rounding to bfloat16 took off O, in bfloat16: see attn_rest_at
    AttnBias bias;
    float* dbias_part;     // [head][padded rows / 64][2·max_distance + 1]
    int64_t dbias_slots;
    float* dkv_part;       // heads of a group in parts: [part][dk, dv][key head][padded row][DP]
    int64_t dkv_rows;      // padded rows of keys
    int32_t dkv_parts;
    int32_t* uneven;       // set by a workgroup of the keys' gradients that meets an uneven tile
    float* part;           // split keys: [split][head][padded row][DP] of O, then of m, l
    float* part_ml;
    int64_t part_rows;
    int32_t splits;
    int32_t heads, kv_heads, dim, dtype, causal;
    int64_t tiles;         // of the uniform plan
    float scale2, scale;   // scale·log2 e, scale
    bool vec_out, vec_q, vec_kv;  // four features of out, dq, dk and dv in one store
};

// A plane of a tile: 64 rows of DP float16 elements, 16-byte pieces permuted so
// that the 16 lanes of an LDS pass meet all banks once, both where they read one
// piece of 16 consecutive rows (along) and where they read 64 bytes of each of
// four rows (across, the transposing read).
template <int DB>
struct AttnTile {
    static constexpr int DP = 32 * DB, kPieces = DP / 8, kRowBytes = 2 * DP;
    static constexpr int kPlane = kAttnRows * kRowBytes;
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (DB == 4) return ((row & 3) << 2) | ((row >> 2) & 3);
        else if constexpr (DB == 2) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else return (row >> 2) & 3;
    }
};

// Operand fragments with their parts, and their product.
template <bool SPLIT>
struct AttnPair {
    f16x8 f[SPLIT ? 2 : 1];
};
__device__ __forceinline__ f32x16 attn_mfma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <bool SPLIT>
__device__ __forceinline__ f32x16 attn_dot(const AttnPair<SPLIT>& a, const AttnPair<SPLIT>& b,
                                           f32x16 c) {
    if constexpr (SPLIT) {
        c = attn_mfma(a.f[1], b.f[0], c);
        c = attn_mfma(a.f[0], b.f[1], c);
    }
    return attn_mfma(a.f[0], b.f[0], c);
}

// The same with the products of the small parts in a sum of their own.
__device__ __forceinline__ f32x16 attn_dot_apart(const AttnPair<true>& a, const AttnPair<true>& b,
                                                 f32x16 c, f32x16& small) {
    small = attn_mfma(a.f[1], b.f[0], small);
    small = attn_mfma(a.f[0], b.f[1], small);
    return attn_mfma(a.f[0], b.f[0], c);
}

// A place in LDS that loads go to directly, as such a pointer from the start: where two
// of them meet in a variable the compiler does not know of which kind a plain one is.
typedef __attribute__((address_space(3))) unsigned char AttnLds;

// Copies bytes of a tile into LDS in pieces of 1 KB, wave by wave.
template <int BYTES>
__device__ __forceinline__ void attn_stage(const char* from, AttnLds* to, int wv, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass emits no stub of a kernel that calls this
    const uint64_t at = reinterpret_cast<uint64_t>(from) + 1024 * wv;
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    const char* base = reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
    static_assert(BYTES % 4096 == 0, "whole pieces for four waves");
#pragma unroll
    for (int i = 0; i < BYTES / 4096; ++i) {
        uint32_t o = 16 * lane;
        asm("" : "+v"(o));  // keeps their sum with the load, whose own it is
        __builtin_amdgcn_global_load_lds(base + 4096 * i + o, to + 1024 * wv + 4096 * i, 16, 0,
                                         0);
    }
#endif
}

// Reads of a staged tile by one lane. along: row l % 32 of a block of 32 rows,
// features 16 ks + 8 (l / 32) ...: the rows are the product's. across: feature
// 32 fb + l % 32, rows 16 s + 8 (j / 4) + 4 (l / 32) + j % 4 for j = 0..7 of a
// block of 32: the rows are summed over, in the order in which a lane holds them
// in a product's result (register 8 s + j), so that a result goes into the next
// product from the registers that it is in. The permutation only flips bits of
// the piece: one lane offset serves all reads of a kind, less an exclusive or.
template <bool SPLIT, int DB>
struct AttnReads {
    using T = AttnTile<DB>;
    int to_along, to_across;
    __device__ __forceinline__ explicit AttnReads(int lane) {
        const int r = lane & 31, i = lane & 15, ar = 4 * (lane >> 5) + (i >> 2);
        to_along = r * T::kRowBytes + 16 * ((lane >> 5) ^ T::swz(r));
        to_across = ar * T::kRowBytes +
                    16 * ((2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ T::swz(ar)) + 8 * (i & 1);
    }
    // PLANE: bytes between the parts, those of a tile or of a stage of fewer rows
    template <int PLANE = T::kPlane>
    __device__ __forceinline__ AttnPair<SPLIT> along(const unsigned char* buf, int b,
                                                     int ks) const {
        AttnPair<SPLIT> r;
#pragma unroll
        for (int p = 0; p < (SPLIT ? 2 : 1); ++p)
            r.f[p] = *reinterpret_cast<const f16x8*>(buf + (to_along ^ (32 * ks)) + p * PLANE +
                                                     32 * b * T::kRowBytes);
        return r;
    }
    template <int PLANE = T::kPlane>
    __device__ __forceinline__ AttnPair<SPLIT> across(const unsigned char* buf, int b, int s,
                                                      int fb) const {
        AttnPair<SPLIT> r;
#pragma unroll
        for (int p = 0; p < (SPLIT ? 2 : 1); ++p) {
            i16x4 x[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
                x[u] = read_turned(buf + (to_across ^ (64 * fb) ^ (32 * u)) + p * PLANE +
                                   (32 * b + 16 * s + 8 * u) * T::kRowBytes);
            r.f[p] = __builtin_bit_cast(
                f16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return r;
    }
};

// Eight results of a lane as an operand: 11 bits, or 22 in two parts.
template <bool SPLIT>
__device__ __forceinline__ AttnPair<SPLIT> attn_operand(const float* x) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    AttnPair<SPLIT> r;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const f32x2 v = {x[j], x[j + 1]};
        const f16x2 h = __builtin_convertvector(v, f16x2);
        r.f[0][j] = h[0];
        r.f[0][j + 1] = h[1];
        if constexpr (SPLIT) {
            const f32x2 d = {x[j] - static_cast<float>(h[0]), x[j + 1] - static_cast<float>(h[1])};
            const f16x2 l = __builtin_convertvector(d, f16x2);
            r.f[1][j] = l[0];
            r.f[1][j + 1] = l[1];
        }
    }
    return r;
}

// N steps of a read from LDS and its use in a product, the reads D steps ahead: left
// to itself the compiler puts each read right before its use, and the matrix
// cores wait for the LDS at every step.
template <bool SPLIT, int N, int D, class Read, class Use>
__device__ __forceinline__ void attn_pipeline(Read&& read, Use&& use) {
    AttnPair<SPLIT> f[D];
    static_for<(D < N ? D : N)>([&](auto i) { f[i.value] = read(i); });
    __builtin_amdgcn_sched_barrier(0);
    static_for<N>([&](auto i) {
        use(i, f[i.value % D]);
        if constexpr (i.value + D < N) {
            f[i.value % D] = read(std::integral_constant<int, i.value + D>{});
            __builtin_amdgcn_sched_barrier(0);
        }
    });
}
template <bool SPLIT>
constexpr int kAttnAhead = SPLIT ? 2 : 4;

// acc[fb] += X^T·W over NB blocks of 32 staged rows X, W a lane's 16 results of
// each (zero where the pair is masked) as operands.
template <bool SPLIT, int DB, int NB, int PLANE = AttnTile<DB>::kPlane>
__device__ __forceinline__ void attn_accumulate(const AttnReads<SPLIT, DB>& rd,
                                                const unsigned char* buf, int b0,
                                                const AttnPair<SPLIT> (&w)[NB][2],
                                                f32x16 (&acc)[DB]) {
    attn_pipeline<SPLIT, 2 * NB * DB, kAttnAhead<SPLIT>>(
        [&](auto i) __attribute__((always_inline)) {
            constexpr int fb = i.value % DB, s = i.value / DB % 2, b = i.value / DB / 2;
            return rd.template across<PLANE>(buf, b0 + b, s, fb);
        },
        [&](auto i, const AttnPair<SPLIT>& x) __attribute__((always_inline)) {
            constexpr int fb = i.value % DB, s = i.value / DB % 2, b = i.value / DB / 2;
            acc[fb] = attn_dot<SPLIT>(x, w[b][s], acc[fb]);
        });
}

// Row (in a block of 32) that register r of a result belongs to.
__device__ __forceinline__ int attn_row(int r, int lane) {
    return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

// Where O's rests of a padded row (of all heads) and a feature lie: for 32 rows and
// eight features as the lanes of a wave hold them, four each, in one piece. (Row by
// row the forward took 61 us at 8191 packed tokens, 16 heads of 128, so 57.)
__device__ __forceinline__ int64_t attn_rest_at(int64_t row, int f, int dp) {
    return (row / 32 * (dp / 8) + f / 8) * 256 + (f / 4 & 1) * 128 + (row & 31) * 4 + (f & 3);
}

__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^e for any e; 0 below the smallest.
__device__ __forceinline__ float attn_pow2(int e) { return ldexpf(1.0f, e); }

// A value at an address that is the same for the whole wave, by a scalar load: a
// vector load's wait would be for the tiles on their way into LDS before it too
// (vector loads return in order), and undo their reading ahead. Of memory that the
// kernel does not write.
template <class V>
__device__ __forceinline__ V attn_scalar(const V* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    return *reinterpret_cast<const __attribute__((address_space(4))) V*>(
        static_cast<uint64_t>(hi) << 32 | lo);
#else
    return *p;
#endif
}

// Exponent of a tile of an operand.
__device__ __forceinline__ int attn_exp(const AttnOp& op, int head, int64_t padded_row) {
    return attn_scalar(op.exps + head * op.exps_sh + (padded_row >> 6)) >> 2;
}

// A lane's share of the flags of an operand's tiles [t0, t1), of which there is one: of the
// first 64, by a load without a branch, so that several operands' are on their way together,
// and of the rest. Then whether one of the shares, of any lane, is of an uneven tile.
__device__ __forceinline__ int attn_flags(const AttnOp& op, int head, int64_t t0, int64_t t1,
                                          int lane) {
    const int64_t i = t0 + lane;
    return op.exps[head * op.exps_sh + (i < t1 ? i : t1 - 1)];
}
__device__ __forceinline__ int attn_more_flags(const AttnOp& op, int head, int64_t t0, int64_t t1,
                                               int lane) {
    int any = 0;
    for (int64_t i = t0 + kWave + lane; i < t1; i += kWave) any |= op.exps[head * op.exps_sh + i];
    return any;
}
__device__ __forceinline__ bool attn_uneven(int flags) {
    return __builtin_amdgcn_ballot_w64((flags & 2) != 0) != 0;
}

// Exponents of four consecutive rows, and one of them.
__device__ __forceinline__ uint32_t attn_four_rows(const int8_t* p) {
    return *reinterpret_cast<const uint32_t*>(p);
}
__device__ __forceinline__ int attn_one_of(uint32_t four, int j) {
    return static_cast<int>(four << (24 - 8 * j)) >> 24;
}

// Exponent of a value that is not 0.
__device__ __forceinline__ int attn_exponent(float x) {
    return static_cast<int>(__float_as_uint(x) >> 23 & 0xff) - 127;
}

// The bias of a distance (query - key) of one head, times log2 e. Buckets are
// counted rather than searched: their starts then come by scalar loads.
__device__ __forceinline__ float attn_bias_of(const AttnBias& b, int heads, int head, int away) {
    const int one = b.one_sided ? b.buckets : b.buckets / 2, n = away < 0 ? -away : away;
    int bucket = -1;
    for (int k = 0; k < one; ++k) bucket += b.starts[k] <= n ? 1 : 0;
    if (!b.one_sided && away < 0) bucket += one;
    const int64_t at = static_cast<int64_t>(bucket) * heads + head;
    const float x = b.dtype == SLK_F32 ? static_cast<const float*>(b.table)[at]
                                       : bf16_to_f32(static_cast<const uint16_t*>(b.table)[at]);
    // a finite one stays finite: a bias of the type's lowest value outweighs the others,
    // it does not hide a key whose row has no other
    const float y = x * kLog2e;
    return fabsf(x) < INFINITY ? fminf(fmaxf(y, -3e38f), 3e38f) : y;
}

// A head's biases into LDS (all threads; a barrier follows), the last ones on both
// sides repeated so far that a block of 32 x 32 with a pair nearer than
// max_distance needs no clamping: distance d at row[max_distance + kAttnFar + d].
constexpr int kAttnFar = 64;
__host__ __device__ constexpr int attn_bias_floats(int md) { return 2 * (md + kAttnFar) + 1; }
__device__ __forceinline__ void attn_bias_row(const AttnBias& b, int head, float* row) {
    const int md = b.max_distance;
    const float* from = b.rows + static_cast<int64_t>(head) * (2 * md + 1) + md;
    for (int i = threadIdx.x; i < attn_bias_floats(md); i += blockDim.x) {
        const int d = i - md - kAttnFar;
        row[i] = from[d < -md ? -md : d > md ? md : d];
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
