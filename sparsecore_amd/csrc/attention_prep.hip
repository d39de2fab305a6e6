// What comes before the attention kernels: the sequences' table and tile order,
// operands in 16-bit parts, and the backward's row sums of dO∘O.
#include "attention.hpp"
#include "attention_prep.hpp"
#include "elem.hpp"

namespace slk {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kBins = 1024;  // classes of work in the tile order
static_assert(kBins == kPlanThreads, "a thread a class");
constexpr int kTileRows = kAttnTileRows;

// Inclusive scan over the workgroup, by sum or maximum, and its last value.
template <bool MAX>
__device__ int64_t scan(int64_t x, int64_t* lds, int64_t& last) {
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    auto both = [](int64_t a, int64_t b) { return MAX ? (a > b ? a : b) : a + b; };
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x = both(x, y);
    }
    __syncthreads();  // lds may still be read
    if (lane == 63) lds[wv] = x;
    __syncthreads();
    int64_t before = MAX ? INT64_MIN : 0, all = before;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w == wv) before = all;
        all = both(all, lds[w]);
    }
    last = all;
    return wv == 0 ? x : both(before, x);
}

// One workgroup, as each sequence's place follows from those before it: 10 us for 23
// sequences of 8191 tokens, its loads and barriers one after the other (16 with a
// thread for all tiles of a sequence). Offsets that fall, or pass the arrays' end, are
// taken as the nearest ones that do not: no row is written twice or outside.
__global__ __launch_bounds__(kPlanThreads) void attn_plan_kernel(const AttnPlanArgs a) {
    __shared__ int64_t lds[kPlanThreads / 64], ends[2];
    __shared__ int32_t bin[kBins];
    const int t = threadIdx.x;
    const bool packed = a.q_offsets != nullptr;
    int64_t pq = 0, pk = 0, endq = 0, endk = 0;
    for (int64_t s0 = 0; s0 < a.n; s0 += kPlanThreads) {
        const int64_t s = s0 + t;
        const bool in = s < a.n;
        AttnSeq x{};
        if (packed) {
            auto clamp = [](int64_t v, int64_t hi) { return v < 0 ? 0 : v > hi ? hi : v; };
            const int64_t oq = in ? clamp(a.q_offsets[s], a.rows_q) : a.rows_q;
            const int64_t ok = in ? clamp(a.k_offsets[s], a.rows_k) : a.rows_k;
            const int64_t nq = in ? clamp(a.q_offsets[s + 1], a.rows_q) : a.rows_q;
            const int64_t nk = in ? clamp(a.k_offsets[s + 1], a.rows_k) : a.rows_k;
            int64_t bq = oq, bk = ok;
            // starts are the running maximum of the offsets: themselves if none falls
            if (!__syncthreads_and(nq >= oq && nk >= ok && oq >= endq && ok >= endk)) {
                int64_t last;
                bq = scan<true>(oq, lds, last);
                bk = scan<true>(ok, lds, last);
                bq = bq > endq ? bq : endq;
                bk = bk > endk ? bk : endk;
            }
            x.q0 = static_cast<int32_t>(bq);
            x.k0 = static_cast<int32_t>(bk);
            x.nq = x.eq = static_cast<int32_t>(in && nq > bq ? nq - bq : 0);
            x.nk = x.ek = static_cast<int32_t>(in && nk > bk ? nk - bk : 0);
            if (in && (t == kPlanThreads - 1 || s == a.n - 1)) {
                ends[0] = bq + x.nq;
                ends[1] = bk + x.nk;
            }
            __syncthreads();
            endq = ends[0];
            endk = ends[1];
        } else {
            auto live = [&](const int32_t* p, int64_t rows) {
                const int64_t n = p != nullptr ? p[s] : rows;
                return static_cast<int32_t>(n < 0 ? 0 : n > rows ? rows : n);
            };
            x.nq = in ? live(a.q_lengths, a.rows_q) : 0;
            x.nk = in ? live(a.k_lengths, a.rows_k) : 0;
            x.eq = static_cast<int32_t>(a.rows_q);
            x.ek = static_cast<int32_t>(a.rows_k);
        }
        const int64_t wq = in ? ceil_div(x.nq, kAttnRows) * kAttnRows : 0;
        const int64_t wk = in ? ceil_div(x.nk, kAttnRows) * kAttnRows : 0;
        int64_t both;  // sums of queries' and keys' rows, each below 2^31
        const int64_t upto = scan<false>(wq << 32 | wk, lds, both);
        const int64_t iq = upto >> 32, ik = upto & 0xffffffff;
        const int64_t totq = both >> 32, totk = both & 0xffffffff;
        x.pq = static_cast<int32_t>(pq + iq - wq);
        x.pk = static_cast<int32_t>(pk + ik - wk);
        pq += totq;
        pk += totk;
        if (in) a.seqs[s] = x;
    }
    if (t == 0 && packed) {
        // rows of no sequence, before the first and behind the last: written as zeros
        int64_t fq = a.q_offsets[0], fk = a.k_offsets[0];
        fq = fq < 0 ? 0 : fq > a.rows_q ? a.rows_q : fq;
        fk = fk < 0 ? 0 : fk > a.rows_k ? a.rows_k : fk;
        AttnSeq x{};
        x.pq = static_cast<int32_t>(pq);
        x.pk = static_cast<int32_t>(pk);
        x.eq = static_cast<int32_t>(fq);
        x.ek = static_cast<int32_t>(fk);
        a.seqs[a.n] = x;
        if (a.n == 0) endq = fq, endk = fk;
        x.q0 = static_cast<int32_t>(endq);
        x.k0 = static_cast<int32_t>(endk);
        x.eq = static_cast<int32_t>(a.rows_q - endq);
        x.ek = static_cast<int32_t>(a.rows_k - endk);
        a.seqs[a.n + 1] = x;
    }
    if (t == 0) {
        a.count[1] = static_cast<int32_t>(pq);
        a.count[3] = static_cast<int32_t>(pk);
    }
    __threadfence_block();
    __syncthreads();
    // tiles by falling work, counted in classes of blocks of 64 on the other side
    const int total = static_cast<int>(a.n) + (packed ? 2 : 0);
    // threads of a sequence, over its tiles; one that has only one sequence keeps it
    int team = 1;
    while (team < 64 && 2 * team * total <= kPlanThreads) team *= 2;
    const int first_s = t / team, at = t % team, step = kPlanThreads / team;
    const bool one_each = total <= step;
    const AttnSeq own = one_each && first_s < total ? a.seqs[first_s] : AttnSeq{};
    for (int side = 0; side < 2; ++side) {
        // the map from tiles of 64 padded rows to sequences, -1 past the last one's
        int32_t* const map = side ? a.k_map : a.q_map;
        const int64_t have = a.count[2 * side + 1] / kAttnRows;
        for (int64_t i = have + t; i < (side ? a.k_tiles : a.q_tiles); i += kPlanThreads)
            map[i] = -1;
        for (int s = first_s; s < static_cast<int>(a.n); s += step) {
            const AttnSeq x = one_each ? own : a.seqs[s];
            const int first = (side ? x.pk : x.pq) / kAttnRows;
            const int tiles = ((side ? x.nk : x.nq) + kAttnRows - 1) / kAttnRows;
            for (int i = at; i < tiles; i += team) map[first + i] = s;
        }
        int2* list = side ? a.k_list : a.q_list;
        if (list == nullptr) continue;
        auto each = [&](auto&& f) {
            for (int s = first_s; s < total; s += step) {
                const AttnSeq x = one_each ? own : a.seqs[s];
                const int shift = x.nk - x.nq;
                const int tiles = ((side ? x.ek : x.eq) + kTileRows - 1) / kTileRows;
                for (int i = at; i < tiles; i += team) {
                    int w;
                    if (side) {
                        w = x.nk <= i * kTileRows ? 0
                            : a.causal            ? x.nq - max(0, i * kTileRows - shift)
                                                  : x.nq;
                    } else {
                        w = x.nq <= i * kTileRows ? 0
                            : a.causal ? min(x.nk, min((i + 1) * kTileRows, x.nq) + shift)
                                       : x.nk;
                    }
                    w = ((max(w, 0) + kAttnRows - 1) / kAttnRows) >> a.work_shift;
                    f(kBins - 1 - min(w, kBins - 1), s, i);
                }
            }
        };
        bin[t] = 0;
        __syncthreads();
        each([&](int b, int, int) { atomicAdd(&bin[b], 1); });
        __syncthreads();
        const int64_t mine = bin[t];
        int64_t all;
        const int64_t upto = scan<false>(mine, lds, all);
        bin[t] = static_cast<int32_t>(upto - mine);
        __syncthreads();
        // the order inside a class does not change a result: tiles are independent
        each([&](int b, int s, int i) { list[atomicAdd(&bin[b], 1)] = int2{s, i}; });
        if (t == 0) a.count[2 * side] = static_cast<int32_t>(all);
        __syncthreads();
    }
}

// A tile of 64 rows x DP features of a tensor in registers. BY_ROWS, for tensors
// whose rows are consecutive in memory: four rows of one feature a piece; else
// eight features of one row. All loads are issued before the first value is
// used: a loop that used each as it came took its memory latency sixteen times
// over (15 us where the bytes take 4).
template <class IO, int DP, bool BY_ROWS>
struct TileRegs {
    static constexpr int kWide = BY_ROWS ? 4 : 8;
    static constexpr int kPer = kAttnRows * DP / kWide / kAttnThreads;
    float v[kPer][kWide];
    // Element j of piece k: row and feature.
    static __device__ __forceinline__ void place(int k, int j, int& r, int& f) {
        const int i = threadIdx.x + kAttnThreads * k;
        if constexpr (BY_ROWS) {
            r = 4 * (i % (kAttnRows / 4)) + j;
            f = i / (kAttnRows / 4);
        } else {
            r = i / (DP / 8);
            f = 8 * (i % (DP / 8)) + j;
        }
    }
    // `at`: the first element; `row`: its row in the tensor (four rows are loaded at
    // once where it is a multiple of four and vec says that the rest is). Pieces past
    // the last row or feature load the first instead: no branch, within which a load's
    // conversion would have to wait for it.
    __device__ __forceinline__ void load(const AttnIo& x, int64_t at, int64_t row, int live,
                                         int dim, int vec) {
        auto clear = [&](int k, int h, int n) {
#pragma unroll
            for (int j = 0; j < n; ++j) v[k][h + j] = 0.0f;
        };
        if (live <= 0) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) clear(k, 0, kWide);
            return;
        }
        if constexpr (!BY_ROWS && IO::kBytes == 2) {
            if (vec == kVecEight) {
                uint4 raw[kPer];
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    int r, f;
                    place(k, 0, r, f);
                    raw[k] = *reinterpret_cast<const uint4*>(
                        x.p + 2 * (at + (r < live ? r : 0) * x.sr + (f < dim ? f : 0)));
                }
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    int r, f;
                    place(k, 0, r, f);
                    const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[k][2 * j] = bf16_to_f32(w[j] & 0xffffu);
                        v[k][2 * j + 1] = bf16_to_f32(w[j] >> 16);
                    }
                    if (r >= live || f >= dim) clear(k, 0, kWide);
                }
                return;
            }
        }
        const bool four = BY_ROWS ? vec == kVecRows && ((row | live) & 3) == 0
                                  : vec == kVecFeatures || vec == kVecEight;
        if (four) {
            using Raw = std::conditional_t<IO::kBytes == 4, f32x4, uint2>;
            Raw raw[kPer][kWide / 4];
#pragma unroll
            for (int k = 0; k < kPer; ++k)
#pragma unroll
                for (int h = 0; h < kWide; h += 4) {
                    int r, f;
                    place(k, h, r, f);
                    raw[k][h / 4] = *reinterpret_cast<const Raw*>(
                        x.p + IO::kBytes * (at + (r < live ? r : 0) * x.sr +
                                            (f < dim ? f : 0) * x.sd));
                }
#pragma unroll
            for (int k = 0; k < kPer; ++k)
#pragma unroll
                for (int h = 0; h < kWide; h += 4) {
                    int r, f;
                    place(k, h, r, f);
                    IO::load4(&raw[k][h / 4], 0, v[k] + h);
                    if (r >= live || f >= dim) clear(k, h, 4);
                }
            return;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k)
#pragma unroll
            for (int j = 0; j < kWide; ++j) {
                int r, f;
                place(k, j, r, f);
                v[k][j] = r < live && f < dim ? IO::load(x.p, at + r * x.sr + f * x.sd) : 0.0f;
            }
    }
};

// Largest of the workgroup's values (bits of non-negative floats) in every thread.
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* lds) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(m, s)));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
    __syncthreads();
    return max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}

__device__ __forceinline__ int tile_exponent(uint32_t top) {
    return max(static_cast<int>(top >> 23) - 127, -100);
}

// Maximum over aligned groups of L lanes, in every lane.
template <int L>
__device__ __forceinline__ uint32_t lane_max(uint32_t m) {
    auto dpp = [&](auto ctrl) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
            0, static_cast<int>(m), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    m = max(m, dpp(std::integral_constant<int, 0xb1>{}));                         // lanes 1, 0, 3, 2
    m = max(m, dpp(std::integral_constant<int, 0x4e>{}));                         // 2, 3, 0, 1
    if constexpr (L >= 8) m = max(m, dpp(std::integral_constant<int, 0x141>{}));  // half-row mirror
    if constexpr (L >= 16) m = max(m, dpp(std::integral_constant<int, 0x140>{})); // row mirror
    if constexpr (L >= 32) m = max(m, static_cast<uint32_t>(__shfl_xor(m, 16)));
    if constexpr (L >= 64) m = max(m, static_cast<uint32_t>(__shfl_xor(m, 32)));
    return m;
}

// Packs a tile of 64 rows of one head: blockIdx.x the tile, blockIdx.y the head of
// an operand; one more y for the rows of biases, a head each. Of dO (with delta
// given) also delta, from the same tile and O's. Rows of consecutive features go
// from registers to their place; consecutive rows are turned through LDS. What
// bounds it is memory: 16384 tokens, 48 heads of 128 in all, bfloat16: 80 us, 5.0
// TB/s (with a branch around each load and eight bytes a load 119); with delta, 32
// heads: 124 us, 4.3 TB/s.
template <bool SPLIT, int DB, class IO, bool DELTA, bool BY_ROWS>
__device__ __forceinline__ void pack_tile(const AttnPack& a, const AttnPackOp& op, int head,
                                          const AttnRow& ro) {
    constexpr int DP = 32 * DB;
    using T = AttnTile<DB>;
    using Regs = TileRegs<IO, DP, BY_ROWS>;
    __shared__ float turn[BY_ROWS ? kAttnRows : 1][BY_ROWS ? DP + 1 : 1];
    __shared__ float sums[DELTA && BY_ROWS ? 16 : 1][kAttnRows];
    __shared__ uint32_t most[4], odd[2];  // odd: rows with a value that is not finite
    __shared__ uint32_t tops[BY_ROWS ? 4 : 1][kAttnRows];  // each row's largest finite magnitude
    const int t = threadIdx.x;
    const int64_t padded = static_cast<int64_t>(blockIdx.x) * kAttnRows;
    const int n = op.keys ? ro.seq.nk : ro.seq.nq, first = op.keys ? ro.seq.k0 : ro.seq.q0;
    const int live = min(max(n - ro.row, 0), kAttnRows);
    const int64_t row = first + ro.row;
    Regs in, out;
    in.load(op.src, ro.sid * op.src.sb + row * op.src.sr + head * op.src.sh, row, live, a.dim,
            op.vec);
    // O in the same pieces as dO, whatever its own order
    if constexpr (DELTA)
        out.load(a.o, ro.sid * a.o.sb + row * a.o.sr + head * a.o.sh, row, live, a.dim, a.o_vec);
    if (DELTA && IO::kBytes == 2 && live > 0) {
        // delta from O before it was rounded: dP - delta cancels, most so in rows that
        // see few keys.
        const int64_t top = head * a.delta_sh + padded;
#pragma unroll
        for (int k = 0; k < Regs::kPer; ++k)
#pragma unroll
            for (int h = 0; h < Regs::kWide; h += 4) {
                int r, f;
                Regs::place(k, h, r, f);
                float x[4];
                if constexpr (BY_ROWS) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[j] = IO::load(a.o_rest,
                                        attn_rest_at(top + (r + j < live ? r + j : 0), f, DP));
                } else {
                    IO::load4(a.o_rest, attn_rest_at(top + (r < live ? r : 0), f, DP), x);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    out.v[k][h + j] += r + (BY_ROWS ? j : 0) < live ? x[j] : 0.0f;
            }
    }
    if (t < 2) odd[t] = 0;
    __syncthreads();
    float d[Regs::kWide];  // BY_ROWS: a thread's share of four rows' delta
#pragma unroll
    for (int j = 0; j < Regs::kWide; ++j) d[j] = 0.0f;
    float rows_d[Regs::kPer];
    uint32_t m[BY_ROWS ? 4 : 1];
#pragma unroll
    for (uint32_t& x : m) x = 0;
#pragma unroll
    for (int k = 0; k < Regs::kPer; ++k) {
        rows_d[k] = 0.0f;
        if constexpr (!BY_ROWS) m[0] = 0;
#pragma unroll
        for (int j = 0; j < Regs::kWide; ++j) {
            int r, f;
            Regs::place(k, j, r, f);
            float& v = in.v[k][j];
            if constexpr (DELTA) {
                if constexpr (BY_ROWS) d[j] = __builtin_fmaf(v, out.v[k][j], d[j]);
                else rows_d[k] = __builtin_fmaf(v, out.v[k][j], rows_d[k]);
            }
            const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
            if (b < 0x7f800000u) {
                m[BY_ROWS ? j : 0] = max(m[BY_ROWS ? j : 0], b);
            } else {
                v = 0.0f;
                atomicOr(&odd[r >> 5], 1u << (r & 31));
            }
            if constexpr (BY_ROWS) turn[r][f] = v;
        }
        if constexpr (!BY_ROWS) {
            const uint32_t top = lane_max<DP / 8>(m[0]);
            int r, f;
            Regs::place(k, 0, r, f);
            if (f == 0) tops[0][r] = top;
        }
    }
    if constexpr (BY_ROWS) {
        // sixteen threads share four rows: every sixteenth of a wave, in four waves
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] = max(m[j], static_cast<uint32_t>(__shfl_xor(m[j], 16)));
            m[j] = max(m[j], static_cast<uint32_t>(__shfl_xor(m[j], 32)));
            if ((t & 63) < 16) tops[t >> 6][4 * (t & 15) + j] = m[j];
        }
    }
    __syncthreads();
    // a lane a row, in every wave
    const int lane = t & 63;
    uint32_t top = tops[0][lane];
    if constexpr (BY_ROWS) top = max(max(top, tops[1][lane]), max(tops[2][lane], tops[3][lane]));
    const int e = tile_exponent(lane_max<64>(top));
    const int own = tile_exponent(top);
    const bool uneven = __builtin_amdgcn_ballot_w64(top != 0 && own < e - kAttnSpread) != 0;
    const int row_e = uneven ? own : e;
    const uint64_t bad = static_cast<uint64_t>(odd[1]) << 32 | odd[0];
    if (t < kAttnRows) op.row_exps[head * op.exps_sh * kAttnRows + padded + t] = row_e;
    if (t == 0) {
        op.exps[head * op.exps_sh + padded / kAttnRows] =
            4 * e + (uneven ? 2 : 0) + (bad != 0 ? 1 : 0);
        op.bad[head * op.exps_sh + padded / kAttnRows] = bad;
    }

    // rows in pieces of eight features, permuted as they will lie in LDS
    const float even = ldexpf(1.0f, kAttnUnit - e);
    char* const to = op.dst + head * op.dst_sh +
                     static_cast<int64_t>(blockIdx.x) * ((SPLIT ? 2 : 1) * T::kPlane);
#pragma unroll
    for (int k = 0; k < kAttnRows * T::kPieces / kAttnThreads; ++k) {
        const int i = kAttnThreads * k + t, r = i / T::kPieces, c = i % T::kPieces;
        const float factor = uneven ? ldexpf(1.0f, kAttnUnit - __shfl(row_e, r)) : even;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (BY_ROWS) v[j] = turn[r][8 * c + j] * factor;
            else v[j] = in.v[k][j] * factor;
        }
        const AttnPair<SPLIT> f = attn_operand<SPLIT>(v);
        char* const at = to + r * T::kRowBytes + 16 * (c ^ T::swz(r));
        *reinterpret_cast<f16x8*>(at) = f.f[0];
        if constexpr (SPLIT) *reinterpret_cast<f16x8*>(at + T::kPlane) = f.f[1];
    }

    if constexpr (DELTA) {
        const int64_t at = head * a.delta_sh + padded;
        uint32_t largest = 0;
        auto put = [&](int r, float y) {
            a.delta[at + r] = y;
            a.lse_out[at + r] = (bad >> r) & 1 ? __builtin_nanf("") : a.lse[at + r];
            const uint32_t b = __float_as_uint(y) & 0x7fffffffu;
            if (b < 0x7f800000u) largest = max(largest, b);
        };
        if constexpr (BY_ROWS) {
            // a thread's four rows are the same in every piece; sixteen threads share them
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[t / 16][4 * (t % 16) + j] = d[j];
            __syncthreads();
            if (t < kAttnRows) {
                float y = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) y += sums[i][t];
                put(t, y);
            }
        } else {
#pragma unroll
            for (int k = 0; k < Regs::kPer; ++k) {
                float y = rows_d[k];
#pragma unroll
                for (int s = 1; s < DP / 8; s <<= 1) y += __shfl_xor(y, s);
                int r, f;
                Regs::place(k, 0, r, f);
                if (f == 0) put(r, y);
            }
        }
        if (t == 0 && blockIdx.x == 0 && head == 0) *a.clear = 0;
        const int de = tile_exponent(block_max(largest, most));
        if (t == 0) a.dexps[head * op.exps_sh + padded / kAttnRows] = de;
    }
}

template <bool SPLIT, int DB, class IO, bool DELTA>
__global__ __launch_bounds__(kAttnThreads) void attn_pack_kernel(const AttnPack a) {
    int which = 0, head = blockIdx.y;
    while (which < a.n && head >= a.op[which].heads) head -= a.op[which++].heads;
    if (which == a.n) {
        const int width = 2 * a.bias.max_distance + 1;
        for (int h = blockIdx.x; h < a.heads; h += gridDim.x)
            for (int i = threadIdx.x; i < width; i += kAttnThreads)
                a.bias.rows[static_cast<int64_t>(h) * width + i] =
                    attn_bias_of(a.bias, a.heads, h, i - a.bias.max_distance);
        return;
    }
    const AttnPackOp& op = a.op[which];
    const int64_t padded = static_cast<int64_t>(blockIdx.x) * kAttnRows;
    if (padded >= op.rows) return;
    const AttnRow ro = attn_row_of(a.plan, op.keys, padded);
    if (!ro.any) return;
    if (op.src.sr == 1 && op.src.sd != 1) pack_tile<SPLIT, DB, IO, DELTA, true>(a, op, head, ro);
    else pack_tile<SPLIT, DB, IO, DELTA, false>(a, op, head, ro);
}

template <bool SPLIT, int DB, class IO>
int pack_as(const AttnPack& a, dim3 grid, hipStream_t st) {
    const dim3 wg(kAttnThreads);
    if (a.delta != nullptr)
        hipLaunchKernelGGL((attn_pack_kernel<SPLIT, DB, IO, true>), grid, wg, 0, st, a);
    else hipLaunchKernelGGL((attn_pack_kernel<SPLIT, DB, IO, false>), grid, wg, 0, st, a);
    return check_launch("attention: pack");
}

template <bool SPLIT, class IO>
int pack(const AttnPack& a, int db, dim3 grid, hipStream_t st) {
    return db == 1   ? pack_as<SPLIT, 1, IO>(a, grid, st)
           : db == 2 ? pack_as<SPLIT, 2, IO>(a, grid, st)
                     : pack_as<SPLIT, 4, IO>(a, grid, st);
}

}  // namespace

int attn_launch_plan(const AttnPlanArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(attn_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    return check_launch("attention: plan");
}

int attn_launch_pack(const AttnPack& a, int db, int dtype, hipStream_t st) {
    int64_t rows = 0, heads = a.bias.table != nullptr ? 1 : 0;
    for (int i = 0; i < a.n; ++i) {
        rows = rows > a.op[i].rows ? rows : a.op[i].rows;
        heads += a.op[i].heads;
    }
    if (rows == 0) return SLK_OK;
    if (heads > 65535) return fail(SLK_EINVAL, "attention: too many heads");
    const dim3 grid(static_cast<unsigned>(rows / kAttnRows), static_cast<unsigned>(heads));
    if (dtype == SLK_F32) return pack<true, F32>(a, db, grid, st);
    return pack<false, BF16>(a, db, grid, st);
}

}  // namespace slk
