// The language-model head and its loss without the logits, slk_linear_ce_*:
//   z = h·Wᵀ (n x v),  lse_n = log Σ_v exp(z_nv),  loss_n = lse_n - z_{n,target}
//   dl = (exp(z - lse) - onehot(target))·g_n,  dh = dl·W,  dW = dlᵀ·h
// Logits exist only as tiles in registers. Forward: each tile leaves its tokens'
// running maximum and sum, which a second kernel joins. Backward: a piece of the
// vocabulary at a time, the tiles are computed again, turned into dl in the
// epilogue and written as the operand of the piece's two gradient products, which
// follow. 2·n·v·d operations forward, 6 backward, where keeping the logits would
// take 4 backward and 4 bytes a logit.
//
// Tokens whose target is ignore_index are left out before anything is computed
// (a list of the live tokens is made on the device), so that they cost nothing
// and what their hidden states hold reaches nothing.
//
// Bound by the matrix cores from some hundred tokens on. 8192 x 4096 x 100000
// bfloat16, forward and backward: 21.5 to 22.4 ms, the logits at 1334 TFLOP/s, dhidden's
// and dweight's products at 1305 and 1203 (a large library product: 1388). 4001 x
// 768 x 32000 float32, 3 in 10 tokens ignored: 1.88 to 1.97 ms, 366 + 471 + 400 + 361
// us in the four products (1100 TFLOP/s as float16), 290 in dl's two operands.
//
// Few tokens are bound by reading W, which they do where it lies: 8 x 2048 x
// 80000 at 4.6 TB/s, forward. A small vocabulary goes the same way, tokens and
// vocabulary exchanged: 8192 x 384 x 65 forward in 13 us, backward in 30 + 7,
// bound by the float32 instructions (13 us of both) and the loads they wait for.
#include "elem.hpp"
#include "mma_tile.hpp"

namespace slk {
namespace {

// Float16 operands are scaled by a power of two a row, so that the row's largest
// finite magnitude lies in [2^13, 2^14): one scale for a whole operand let a token
// of 10^8 times the others' magnitude take the others' digits (their losses were off
// by 1e-3). A row that is not summed over gives its power back in the epilogue, a row
// along the sum has it folded into the other factor, dl, whose own rows are scaled
// by the largest term that each then has.
constexpr int kTopExp = 14;

// What forward leaves for backward: the count of the live tokens.
struct Header {
    int32_t live;
    int32_t pad[31];
};

__device__ __forceinline__ int scale_exp(uint32_t top) {
    // top in [2^(e-1), 2^e): x·2^(14-e) is below 2^14; no scaling of zeros
    const int e = static_cast<int>(top >> 23) - 126;
    if (top == 0) return 0;
    const int s = kTopExp - e;
    return s > 126 ? 126 : s;
}
// x·2^e, rounded once, whatever e
__device__ __forceinline__ float scaled(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

// ───────────────────────────── live tokens ─────────────────────────────

// rows[i] = the i-th live token, pos[n] its place or -1, tgt[i] its target (-1
// if it is no row of the vocabulary: its loss is NaN). One workgroup, kListPer
// slabs of consecutive tokens at a time: a token's place is the live tokens of
// the slabs before, of its slab's earlier waves and of its wave's lower lanes.
constexpr int kListThreads = 1024, kListPer = 8, kListWaves = kListThreads / kWave;
__global__ __launch_bounds__(kListThreads) void ce_list_kernel(
    const int64_t* __restrict__ target, int64_t n, int64_t v, int64_t ignore,
    Header* __restrict__ hd, int32_t* __restrict__ rows, int32_t* __restrict__ pos,
    int32_t* __restrict__ tgt) {
    static_assert(kListPer * kListWaves == 2 * kWave, "two counts a lane below");
    __shared__ int counts[kListPer * kListWaves];
    const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x >> 6;
    int base = 0;
    for (int64_t n0 = 0; n0 < n; n0 += kListThreads * kListPer) {
        int64_t t[kListPer];
        uint64_t live[kListPer];
#pragma unroll
        for (int j = 0; j < kListPer; ++j) {
            const int64_t at = n0 + j * kListThreads + threadIdx.x;
            t[j] = at < n ? target[at] : ignore;
        }
#pragma unroll
        for (int j = 0; j < kListPer; ++j) {
            live[j] = __ballot(t[j] != ignore);
            if (lane == 0) counts[j * kListWaves + wv] = __popcll(live[j]);
        }
        __syncthreads();
        // every wave scans all counts: lane l has 2 l and 2 l + 1
        const int a = counts[2 * lane], b = counts[2 * lane + 1];
        int incl = a + b;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int up = __shfl_up(incl, o);
            if (lane >= o) incl += up;
        }
#pragma unroll
        for (int j = 0; j < kListPer; ++j) {
            const int64_t at = n0 + j * kListThreads + threadIdx.x;
            const int k = j * kListWaves + wv;  // this wave's count, half of lane k / 2's
            const int before = __shfl(incl - b - (k & 1 ? 0 : a), k >> 1);
            const int i = base + before + __popcll(live[j] & ((uint64_t{1} << lane) - 1));
            if (at >= n) continue;
            if (t[j] != ignore) {
                rows[i] = static_cast<int32_t>(at);
                tgt[i] = t[j] >= 0 && t[j] < v ? static_cast<int32_t>(t[j]) : -1;
                pos[at] = i;
            } else {
                pos[at] = -1;
            }
        }
        base += __shfl(incl, kWave - 1);
        __syncthreads();
    }
    if (threadIdx.x == 0) hd->live = base;
}

// The power of two of each row's scale, of hidden (live tokens, at their places) and
// weight, float32: a wave a row of either. The rows past the vocabulary that a tile of
// it covers get 0.
template <bool VEC>
__global__ __launch_bounds__(256) void ce_exp_kernel(const float* __restrict__ h, int64_t n,
                                                     const float* __restrict__ w, int64_t v,
                                                     int64_t tiled, int64_t d,
                                                     const int32_t* __restrict__ pos,
                                                     int32_t* __restrict__ hx,
                                                     int32_t* __restrict__ wx) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4;
    auto see = [](uint32_t& m, float x) {
        const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
        if (b < 0x7f800000u) m = max(m, b);
    };
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
         row < n + tiled; row += waves) {
        const bool of_h = row < n;
        if (row >= n + v) {
            if (lane == 0) wx[row - n] = 0;
            continue;
        }
        if (of_h && pos[row] < 0) continue;
        const float* x = of_h ? h + row * d : w + (row - n) * d;
        uint32_t m = 0;
        if (VEC) {
            int64_t e = 4 * lane;
            for (; e + 4 * 3 * kWave < d; e += 4 * 4 * kWave) {
                f32x4 q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q[j] = *reinterpret_cast<const f32x4*>(x + e + 4 * j * kWave);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) see(m, q[j][i]);
            }
            for (; e < d; e += 4 * kWave) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(x + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) see(m, q[i]);
            }
        } else {
            for (int64_t e = lane; e < d; e += kWave) see(m, x[e]);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(m, o)));
        if (lane == 0) (of_h ? hx[pos[row]] : wx[row - n]) = scale_exp(m);
    }
}

// ───────────────────────────── packing ─────────────────────────────

// hi and lo of eight values
__device__ __forceinline__ void split8(const float (&v)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = static_cast<_Float16>(v[j]);
        lo[j] = static_cast<_Float16>(v[j] - static_cast<float>(hi[j]));
    }
}

struct PackArgs {
    const void* src;
    const int32_t* rows;  // source row of each row, NULL: itself
    const int32_t* live;  // rows that count (device), NULL: R
    const int32_t* exps;  // power of two of each row's scale (float32 sources)
    int64_t R, d;
    int64_t out_rows;  // rows that the packed form is laid out for
    char* out;
};

// Eight elements a thread: consecutive threads take a stage of a row, then its
// next rows. The rows up to the next multiple of 64 are zero.
template <class T, bool SPLIT, bool VEC>
__global__ __launch_bounds__(256) void ce_pack_kernel(const PackArgs p) {
    constexpr int K = kStageK<SPLIT>, kParts = K / 8;
    const int64_t R = p.live != nullptr ? *p.live : p.R;
    const int64_t rows = ceil_div(R, 64) * 64;
    // four rows a thread, their loads in flight together
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int part = static_cast<int>(t % kParts);
    const int64_t st = blockIdx.y;
    const int64_t r0 = t / kParts, step = (rows + 3) / 4;
    if (r0 >= step) return;
    const int64_t e = st * K + 8 * part;
    float x[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = r0 + j * step;
        const bool in = r < R;
        const int64_t off = in ? (p.rows != nullptr ? p.rows[r] : r) * p.d + e : 0;
        if (VEC) {
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                if (in && e + k < p.d) {
                    T::load4(p.src, off + k, &x[j][k]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[j][k + i] = 0.0f;
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                x[j][k] = in && e + k < p.d ? T::load(p.src, off + k) : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = r0 + j * step;
        if (r >= rows) break;
        char* to = p.out + (st * p.out_rows + r) * kStageBytes + 16 * part;
        if constexpr (SPLIT) {
            const int scale = r < R ? p.exps[r] : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[j][k] = scaled(x[j][k], scale);
            f16x8 hi, lo;
            split8(x[j], hi, lo);
            *reinterpret_cast<f16x8*>(to) = hi;
            *reinterpret_cast<f16x8*>(to + 64) = lo;
        } else {
            b16x8 b;
#pragma unroll
            for (int k = 0; k < 8; ++k) b[k] = static_cast<__bf16>(x[j][k]);
            *reinterpret_cast<b16x8*>(to) = b;
        }
    }
}

// ───────────────────────────── epilogues ─────────────────────────────

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The logits themselves: each accumulator by its row's and its token's power of two
// (one exponent, so that nothing between overflows), of the wave's columns b.
template <class Tile>
__device__ __forceinline__ void unscale_logits(f32x16 (&acc)[Tile::kNA][2], const Tile& t, int b,
                                               const int32_t* wx, const int32_t* hx) {
    const int64_t tok = t.n0() + t.col(b);
    const int th = tok < t.N ? hx[tok] : 0;
    const int32_t* mine = wx + t.m0() + t.row(0, 0);
#pragma unroll
    for (int a = 0; a < Tile::kNA; ++a) {
        i32x4 e[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            e[q] = *reinterpret_cast<const i32x4*>(mine + 32 * a + 8 * q);
#pragma unroll
        for (int r = 0; r < 16; ++r)
            acc[a][b][r] = scaled(acc[a][b][r], -(e[r >> 2][r & 3] + th));
        __builtin_amdgcn_sched_barrier(0);  // all blocks' exponents at once spilled registers
    }
}

// exp(x) as 2^(x·log2 e): v_exp_f32 is one instruction (1 ulp). The difference from
// the maximum is taken first, so that it rounds relative to itself: with log2 e inside
// a fused multiply-add the product's rounding, half an ulp of the logit, stayed in the
// exponent, and logits beyond 2^32 overflowed it. A token keeps m and 1/s rather than the
// logarithm of its sum: exp(z - m) / s is then as exact as the difference, where a
// rounded logarithm near 20 would put 1e-6 into every entry of the token's softmax; and
// m - z of a token whose target has the largest logit is 0 exactly.
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// (m, s) joined with (m2, s2); an empty part has m = -inf, s = 0. A NaN stays in s.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
    s = (m == -INFINITY ? s : s * exp_(m - base)) + (m2 == -INFINITY ? s2 : s2 * exp_(m2 - base));
    m = top;
}

// Forward: rows are the vocabulary, columns tokens, so that a lane holds half of
// its wave's logits of each of its two tokens and only their maximum and sum
// cross lanes.
template <bool SPLIT>
struct ScoreEpi {
    const int32_t *wx, *hx;  // powers of two of the operands' rows (SPLIT)
    const int32_t* tgt;
    float2* part;  // vocabulary tiles x tokens
    float* zt;
    int64_t n;
    template <class Tile>
    __device__ __forceinline__ void operator()(f32x16 (&acc)[Tile::kNA][2], const Tile& t) const {
        __syncthreads();  // the ring is free
        float2* sh = reinterpret_cast<float2*>(t.lds);  // kWavesM x kBN
        const int rows = static_cast<int>(t.M - t.m0());  // those of this wave that exist
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if constexpr (SPLIT) unscale_logits(acc, t, b, wx, hx);
            const int64_t tok = t.n0() + t.col(b);
            const int64_t want = (tok < t.N ? tgt[tok] : -1) - t.m0();
            const bool here = want >= 0 && want < 32 * Tile::kNA;
            if (__any(here)) {
#pragma unroll
                for (int a = 0; a < Tile::kNA; ++a)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (t.row(a, r) == want) zt[tok] = acc[a][b][r];
            }
            float m = -INFINITY, s = 0.0f;
            if (rows < 32 * Tile::kNA) {  // past the vocabulary
#pragma unroll
                for (int a = 0; a < Tile::kNA; ++a)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (t.row(a, r) >= rows) acc[a][b][r] = -INFINITY;
            }
#pragma unroll
            for (int a = 0; a < Tile::kNA; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[a][b][r]);
            m = fmaxf(m, __shfl_xor(m, 32));
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int a = 0; a < Tile::kNA; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += exp_(acc[a][b][r] - base);
            s += __shfl_xor(s, 32);
            if (t.lane < 32) sh[t.wm * Tile::kBN + 64 * t.wn + t.col(b)] = make_float2(m, s);
        }
        __syncthreads();
        if (threadIdx.x < Tile::kBN) {
            const int64_t tok = t.k0 + threadIdx.x;
            float m = -INFINITY, s = 0.0f;
#pragma unroll
            for (int w = 0; w < Tile::kWavesM; ++w) {
                const float2 x = sh[w * Tile::kBN + threadIdx.x];
                join(m, s, x.x, x.y);
            }
            if (tok < t.N) part[t.i0 / kTileM * n + tok] = make_float2(m, s);
        }
    }
};

// Backward: the same tiles as dl, its rows tokens, zero where the live tokens or the
// vocabulary end inside the tile. bfloat16: times the token's upstream gradient, as an
// operand whose stages run along the piece of the vocabulary.
template <bool SPLIT>
struct DlEpi {
    const int32_t* tgt;
    const float2* norm;  // (m, 1 / s) of each token
    const float* gr;     // upstream gradient of each token, NULL: all 1
    char* out;
    int64_t v0;    // first row of the piece
    int64_t rows;  // tokens that it is laid out for: whole tiles
    template <class Tile>
    __device__ __forceinline__ void operator()(f32x16 (&acc)[Tile::kNA][2], const Tile& t) const {
        const int have = static_cast<int>(t.M - t.m0());  // those rows of this wave that exist
        constexpr int K = kStageK<false>;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t tok = t.n0() + t.col(b);
            const bool in = tok < t.N;
            const int64_t want = (in ? tgt[tok] - v0 : -1) - t.m0();
            const bool any = __any(want >= 0 && want < 32 * Tile::kNA);
            const float2 ms = in ? norm[tok] : make_float2(0.0f, 0.0f);
            const float g = in ? (gr != nullptr ? gr[tok] : 1.0f) : 0.0f;
            const float gs = g * ms.y;
#pragma unroll
            for (int a = 0; a < Tile::kNA; ++a) {
                const int64_t v = t.m0() + 32 * a;  // this block's 32 rows
                char* to = out + ((v / K) * rows + tok) * kStageBytes + 2 * (v % K);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint16_t h[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 4 * q + j;
                        float p = exp_(acc[a][b][r] - ms.x) * gs;
                        if (any && t.row(a, r) == want) p -= g;
                        p = in && t.row(a, r) < have ? p : 0.0f;
                        h[j] = f32_to_bf16(p);
                    }
                    const int at = 2 * (8 * q + 4 * (t.lane >> 5));
                    *reinterpret_cast<ushort4*>(to + at) = make_ushort4(h[0], h[1], h[2], h[3]);
                }
            }
        }
    }
};

// Float32: dl itself, without the upstream gradients, 32 rows of vocabulary a stage
// like the operands that ce_split_kernel makes of it. dl's rows (tokens) in dh = dl·W
// and its columns in dW = dlᵀ·(g h) run over terms of very different sizes: softmax
// entries of 1e-12 beside 1, rows of W and h of any magnitude. So each gets the power
// of two of its own largest term, which this tile's part of is left here: of a token
// max |dl|·2^-wx, of a row of the vocabulary max |dl g|·2^-hx, as exponents. (One array
// of halves for both products, scaled by 2^14, kept 2^-39 of 1 and no more: it took
// neither the second array nor the pass that makes the two, 0.3 of 1.6 ms at 4001 x
// 768 x 32000, and lost the gradient of rows that softmax hardly reaches.)
constexpr int kNoTerm = -(1 << 20);
__device__ __forceinline__ int term_exp(float x, int e) {
    return x == 0.0f ? kNoTerm : __builtin_amdgcn_frexp_expf(x) + e;
}
// the largest of 32 lanes, in lanes 31 and 63
__device__ __forceinline__ int half_max(int x) {
    auto step = [&](auto ctrl, auto rows) {
        constexpr int C = decltype(ctrl)::value, R = decltype(rows)::value;
        x = max(x, __builtin_amdgcn_update_dpp(x, x, C, R, 0xf, false));
    };
    using std::integral_constant;
    step(integral_constant<int, 0xB1>{}, integral_constant<int, 0xf>{});   // lane ^ 1
    step(integral_constant<int, 0x4E>{}, integral_constant<int, 0xf>{});   // lane ^ 2
    step(integral_constant<int, 0x141>{}, integral_constant<int, 0xf>{});  // half row mirrored
    step(integral_constant<int, 0x140>{}, integral_constant<int, 0xf>{});  // row mirrored
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // rows 0, 2 to 1, 3
    return x;
}
template <>
struct DlEpi<true> {
    const int32_t *wx, *hx;  // of the piece's rows, of the tokens
    const int32_t* tgt;
    const float2* norm;
    const float* gr;
    char* out;
    int64_t v0, rows;
    int32_t* row_part;  // tiles of vocabulary x tokens (rows)
    int32_t* col_part;  // tiles of tokens x rows of the piece
    int64_t piece;
    template <class Tile>
    __device__ __forceinline__ void operator()(f32x16 (&acc)[Tile::kNA][2], const Tile& t) const {
        constexpr int kWavesN = Tile::kBN / 64;
        __syncthreads();  // the ring is free
        int* sh_tok = reinterpret_cast<int*>(t.lds);         // kWavesM x kBN
        int* sh_voc = sh_tok + Tile::kWavesM * Tile::kBN;    // kWavesN x kTileM
        const int have = static_cast<int>(t.M - t.m0());  // those rows of this wave that exist
        int want[2], hexp[2], big[2];
        float2 ms[2];
        float g[2];
        bool in[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t tok = t.n0() + t.col(b);
            in[b] = tok < t.N;
            const int64_t row = (in[b] ? tgt[tok] - v0 : -1) - t.m0();
            want[b] = row >= 0 && row < 32 * Tile::kNA ? static_cast<int>(row) : -1;
            ms[b] = in[b] ? norm[tok] : make_float2(0.0f, 0.0f);
            g[b] = in[b] && gr != nullptr ? gr[tok] : 1.0f;
            hexp[b] = in[b] ? -hx[tok] : 0;
            big[b] = kNoTerm;
        }
        const bool any = __any(want[0] >= 0 || want[1] >= 0);
#pragma unroll
        for (int a = 0; a < Tile::kNA; ++a) {
            const int64_t v = t.m0() + 32 * a;  // this block's 32 rows: a stage
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = t.row(a, 4 * q);
                const i32x4 we = *reinterpret_cast<const i32x4*>(wx + t.m0() + row);
                i32x4 most = {kNoTerm, kNoTerm, kNoTerm, kNoTerm};
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    f32x4 x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float z = scaled(acc[a][b][4 * q + j], hexp[b] - we[j]);
                        float p = exp_(z - ms[b].x) * ms[b].y;
                        if (any && row + j == want[b]) p -= 1.0f;
                        p = in[b] && row + j < have ? p : 0.0f;
                        x[j] = p;
                        big[b] = max(big[b], term_exp(p, -we[j]));
                        most[j] = max(most[j], term_exp(p * g[b], hexp[b]));
                    }
                    *reinterpret_cast<f32x4*>(out +
                                              ((v / 32) * rows + t.n0() + t.col(b)) * kStageBytes +
                                              4 * (row - 32 * a)) = x;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) most[j] = half_max(most[j]);
                if ((t.lane & 31) == 31)
                    *reinterpret_cast<i32x4*>(sh_voc + t.wn * kTileM + 32 * Tile::kNA * t.wm +
                                              row) = most;
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int m = max(big[b], __shfl_xor(big[b], 32));
            if (t.lane < 32) sh_tok[t.wm * Tile::kBN + 64 * t.wn + t.col(b)] = m;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < Tile::kBN; i += kMmaThreads) {
            int m = kNoTerm;
#pragma unroll
            for (int w = 0; w < Tile::kWavesM; ++w) m = max(m, sh_tok[w * Tile::kBN + i]);
            row_part[t.i0 / kTileM * rows + t.k0 + i] = m;
        }
        for (int i = threadIdx.x; i < kTileM; i += kMmaThreads) {
            int m = kNoTerm;
#pragma unroll
            for (int w = 0; w < kWavesN; ++w) m = max(m, sh_voc[w * kTileM + i]);
            col_part[t.k0 / Tile::kBN * piece + t.i0 + i] = m;
        }
    }
};

// The powers of two of dl's rows and columns from their tiles' parts: 32 of them a
// workgroup, eight threads each; the tokens' workgroups first.
struct TermArgs {
    const int32_t *row_part, *col_part;
    const int32_t* live;
    int64_t rows, piece, vn;
    int bn;  // tokens of a tile
    int32_t *row_exp, *col_exp;
};
__global__ __launch_bounds__(256) void ce_term_kernel(const TermArgs p) {
    __shared__ int sh[8][32];
    const int64_t live = *p.live, groups = ceil_div(p.rows, 32);
    const bool of_row = blockIdx.x < groups;
    const int64_t i = 32 * (of_row ? blockIdx.x : blockIdx.x - groups) + (threadIdx.x & 31);
    const int part = threadIdx.x >> 5;
    const int64_t width = of_row ? p.rows : p.piece;
    const int64_t parts = of_row ? ceil_div(p.vn, kTileM) : ceil_div(live, p.bn);
    const bool in = of_row ? i < live : i < ceil_div(p.vn, kTileM) * kTileM;
    const int32_t* from = of_row ? p.row_part : p.col_part;
    int m = kNoTerm;
    if (in) {
        for (int64_t k = part; k < parts; k += 8) m = max(m, from[k * width + i]);
    }
    sh[part][threadIdx.x & 31] = m;
    __syncthreads();
    if (part != 0 || i >= width) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) m = max(m, sh[k][threadIdx.x]);
    (of_row ? p.row_exp : p.col_exp)[i] = m == kNoTerm ? 0 : kTopExp - m;
}

// dl as the operands of its two products, scaled as above, in halves: dh's into its
// own array, dW's in dl's place. Eight entries of a token a thread, four tokens.
struct DlArgs {
    char* dl;   // in: float32; out: dW's operand (NULL for neither: not wanted)
    char* dlh;  // dh's operand
    bool of_w;
    const int32_t *wx, *hx, *row_exp, *col_exp;
    const float* gr;  // NULL: all 1
    const int32_t* live;
    int64_t rows;
};
__global__ __launch_bounds__(256) void ce_split_kernel(const DlArgs p) {
    const int64_t rows = ceil_div(static_cast<int64_t>(*p.live), 64) * 64;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int part = static_cast<int>(t & 3);
    const int64_t st = blockIdx.y, r0 = t >> 2, step = rows / 4;
    if (r0 >= step) return;
    const int64_t v = 32 * st + 8 * part;
    int we[8], ce[8];
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(p.wx + v + k);
        const i32x4 b = *reinterpret_cast<const i32x4*>(p.col_exp + v + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            we[k + j] = a[j];
            ce[k + j] = b[j];
        }
    }
    f32x4 x[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const char* from = p.dl + (st * p.rows + r0 + j * step) * kStageBytes + 32 * part;
        x[j][0] = *reinterpret_cast<const f32x4*>(from);
        x[j][1] = *reinterpret_cast<const f32x4*>(from + 16);
    }
    // a row's four threads are neighbours in one wave: what one overwrites below all
    // have loaded above
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = r0 + j * step;
        const int64_t at = (st * p.rows + r) * kStageBytes + 16 * part;
        const bool in = r < *p.live;
        float y[8];
        f16x8 hi, lo;
        if (p.dlh != nullptr) {
            const int re = in ? p.row_exp[r] : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = scaled(x[j][k >> 2][k & 3], re - we[k]);
            split8(y, hi, lo);
            *reinterpret_cast<f16x8*>(p.dlh + at) = hi;
            *reinterpret_cast<f16x8*>(p.dlh + at + 64) = lo;
        }
        if (p.of_w) {
            const int he = in ? p.hx[r] : 0;
            const float g = in && p.gr != nullptr ? p.gr[r] : 1.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = scaled(x[j][k >> 2][k & 3] * g, ce[k] - he);
            split8(y, hi, lo);
            *reinterpret_cast<f16x8*>(p.dl + at) = hi;
            *reinterpret_cast<f16x8*>(p.dl + at + 64) = lo;
        }
    }
}

// The sums of a product whose first operand's rows were scaled: their powers of two
// given back (before anything else, so that this rounds only what is subnormal).
template <class Tile>
__device__ __forceinline__ void unscale_rows(f32x16 (&acc)[2], const Tile& t, int a,
                                             const int32_t* exps) {
    i32x4 e[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        e[q] = *reinterpret_cast<const i32x4*>(exps + t.m0() + t.row(a, 4 * q));
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] = scaled(acc[b][r], -e[r >> 2][r & 3]);
    __builtin_amdgcn_sched_barrier(0);
}

// Gradient products: float32 sums of each part of the K loop.
template <bool SPLIT>
struct SumEpi {
    float* out;  // splits x rows x d
    const int32_t* exps;  // of the first operand's rows (SPLIT)
    int64_t rows, d;
    bool add;  // onto what the vocabulary's earlier pieces left
    template <class Tile>
    __device__ __forceinline__ void operator()(f32x16 (&acc)[Tile::kNA][2], const Tile& t) const {
        float* to = out + t.split * rows * d;
#pragma unroll
        for (int a = 0; a < Tile::kNA; ++a) {
            if constexpr (SPLIT) unscale_rows(acc[a], t, a, exps);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int64_t c = t.n0() + t.col(b);
                if (add) {  // the block's loads in flight together
                    float old[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int64_t row = t.m0() + t.row(a, r);
                        old[r] = row < t.M && c < t.N ? to[row * d + c] : 0.0f;
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[a][b][r] += old[r];
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int64_t row = t.m0() + t.row(a, r);
                    if (row < t.M && c < t.N) to[row * d + c] = acc[a][b][r];
                }
            }
        }
    }
};

// dW where one workgroup has the whole sum: scaled, rounded and stored.
template <class T, bool SPLIT>
struct WeightEpi {
    const int32_t* exps;
    const float* factor;
    void* out;  // of the piece's first row
    int64_t d;
    template <class Tile>
    __device__ __forceinline__ void operator()(f32x16 (&acc)[Tile::kNA][2], const Tile& t) const {
        const float f = *factor;
#pragma unroll
        for (int a = 0; a < Tile::kNA; ++a) {
            if constexpr (SPLIT) unscale_rows(acc[a], t, a, exps);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int64_t c = t.n0() + t.col(b);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int64_t row = t.m0() + t.row(a, r);
                    if (row < t.M && c < t.N) T::store(out, row * d + c, acc[a][b][r] * f);
                }
            }
        }
    }
};

// dh where one workgroup has the whole sum: to the token's row.
template <class T, bool SPLIT>
struct TokenEpi {
    const int32_t* exps;
    const float *factor, *gr;  // gr: each token's own in its place (SPLIT; NULL: none)
    const int32_t* rows;
    void* out;
    int64_t d;
    template <class Tile>
    __device__ __forceinline__ void operator()(f32x16 (&acc)[Tile::kNA][2], const Tile& t) const {
        const float f = *factor;
#pragma unroll
        for (int a = 0; a < Tile::kNA; ++a) {
            if constexpr (SPLIT) unscale_rows(acc[a], t, a, exps);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t row = t.m0() + t.row(a, r);
                if (row >= t.M) continue;
                const int64_t at = rows[row] * d;
                const float g = SPLIT && gr != nullptr ? gr[row] : f;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int64_t c = t.n0() + t.col(b);
                    if (c < t.N) T::store(out, at + c, acc[a][b][r] * g);
                }
            }
        }
    }
};

// ───────────────────────────── joining ─────────────────────────────

// Maximum, sum and loss of each token from its partial maxima and sums: TOK tokens a
// workgroup, 256 / TOK threads a token.
struct JoinArgs {
    const float2* part;
    const float* zt;
    const int64_t* target;
    const int32_t* pos;  // place of each token in part, NULL: its own
    const int32_t* tgt;  // target of each place, -1: none (with pos)
    float2* norm;        // (m, 1 / s) of each place, NULL: not wanted
    float* losses;
    int64_t n, v, ignore, parts;
};
template <int TOK>
__global__ __launch_bounds__(256) void ce_join_kernel(const JoinArgs p) {
    __shared__ float2 sh[4][TOK];
    const int j = threadIdx.x % TOK, part = threadIdx.x / TOK;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * TOK + j;
    int64_t i = -1;
    bool valid = false;
    if (n < p.n) {
        if (p.pos != nullptr) {
            i = p.pos[n];
            valid = i >= 0 && p.tgt[i] >= 0;
        } else if (p.target[n] != p.ignore) {
            i = n;
            valid = p.target[n] >= 0 && p.target[n] < p.v;
        }
    }
    float m = -INFINITY, s = 0.0f;
    if (i >= 0) {
        for (int64_t k = part; k < p.parts; k += 256 / TOK) {
            const float2 x = p.part[k * p.n + i];
            join(m, s, x.x, x.y);
        }
    }
    // lanes TOK apart hold a token's parts: within the wave, then over the four waves
#pragma unroll
    for (int o = TOK; o < kWave; o <<= 1) {
        const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
        join(m, s, m2, s2);
    }
    if ((threadIdx.x & (kWave - 1)) < TOK) sh[threadIdx.x >> 6][j] = make_float2(m, s);
    __syncthreads();
    if (part != 0 || n >= p.n) return;
#pragma unroll
    for (int k = 1; k < 4; ++k) join(m, s, sh[k][j].x, sh[k][j].y);
    if (i < 0) {
        p.losses[n] = 0.0f;
        return;
    }
    if (m == -INFINITY) m = 0.0f;
    if (p.norm != nullptr) p.norm[i] = make_float2(m, 1.0f / s);
    p.losses[n] = valid ? (m - p.zt[i]) + log2f(s) * kLn2 : NAN;
}

// The sum or mean of the losses over the live tokens: one workgroup, sums in
// float64 in a fixed order.
__global__ __launch_bounds__(1024) void ce_reduce_kernel(const float* __restrict__ losses,
                                                         const int64_t* __restrict__ target,
                                                         int64_t n, int64_t ignore, bool mean,
                                                         float* __restrict__ live,
                                                         float* __restrict__ out) {
    __shared__ double sh[2][1024 / kWave];
    double s = 0.0, c = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        s += losses[i];
        c += target[i] != ignore;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        s += __shfl_xor(s, o);
        c += __shfl_xor(c, o);
    }
    if ((threadIdx.x & (kWave - 1)) == 0) {
        sh[0][threadIdx.x >> 6] = s;
        sh[1][threadIdx.x >> 6] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 1024 / kWave; ++w) {
            s += sh[0][w];
            c += sh[1][w];
        }
        *out = static_cast<float>(mean ? s / c : s);  // no live token: 0 / 0
        if (live != nullptr) *live = static_cast<float>(c);
    }
}

// Upstream gradients: factor is the one for all tokens (sum, mean), or gr each live
// token's own (none; factor is 1).
// The workgroups beside the first clear the rows of dh that are no live token's,
// where the product writes only the others.
template <class T>
__global__ __launch_bounds__(1024) void ce_upstream_kernel(
    const float* __restrict__ up, const Header* __restrict__ hd, const int32_t* __restrict__ rows,
    int reduction, float* __restrict__ gr, float* __restrict__ factor,
    const int32_t* __restrict__ pos, int64_t n, int64_t d, void* __restrict__ dh) {
    if (blockIdx.x > 0) {
        const int lane = threadIdx.x & (kWave - 1);
        const int64_t waves = static_cast<int64_t>(gridDim.x - 1) * (1024 / kWave);
        for (int64_t w = static_cast<int64_t>(blockIdx.x - 1) * (1024 / kWave) +
                         (threadIdx.x >> 6);
             w * kWave < n; w += waves) {
            const int64_t mine = w * kWave + lane;
            uint64_t clear = __ballot(mine < n && pos[mine < n ? mine : 0] < 0);
            while (clear != 0) {
                const int64_t row = w * kWave + __ffsll(static_cast<unsigned long long>(clear)) - 1;
                clear &= clear - 1;
                for (int64_t e = lane; e < d; e += kWave) T::store(dh, row * d + e, 0.0f);
            }
        }
        return;
    }
    const int64_t live = hd->live;
    if (reduction == SLK_REDUCE_NONE) {
        for (int64_t i = threadIdx.x; i < live; i += 1024) gr[i] = up[rows[i]];
        if (threadIdx.x == 0) *factor = 1.0f;
    } else if (threadIdx.x == 0) {
        // no live token: gradients are 0, as the sum's over none
        *factor = live == 0 ? 0.0f
                  : reduction == SLK_REDUCE_MEAN ? *up / static_cast<float>(live) : *up;
    }
}

// out[r][c] = the parts' sum times the upstream factor (gr: the token's own), rounded;
// with pos, row r is token r and the sums are at its place (0 where it has none).
template <class T>
__global__ __launch_bounds__(256) void ce_finish_kernel(const float* __restrict__ sums, int splits,
                                                        int64_t rows, int64_t stride, int64_t d,
                                                        const int32_t* __restrict__ pos,
                                                        const float* __restrict__ factor,
                                                        const float* __restrict__ gr,
                                                        void* __restrict__ out) {
    const float f = *factor;
    const int64_t total = rows * d, step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
        const int64_t r = i / d;
        const int64_t at = pos != nullptr ? pos[r] : r;
        float x = 0.0f;
        if (at >= 0) {
            const float* from = sums + at * d + (i - r * d);
            int k = 0;
            for (; k + 8 <= splits; k += 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = from[(k + j) * stride * d];
#pragma unroll
                for (int j = 0; j < 8; ++j) x += v[j];
            }
            for (; k < splits; ++k) x += from[k * stride * d];
            x *= gr != nullptr ? gr[at] : f;
        }
        T::store(out, i, x);
    }
}

// ───────────────────────────── few tokens ─────────────────────────────

// Few tokens read W where it lies, once forward and once backward: its packed
// copy alone would be read and written three times more. Up to how many, by what
// the two ways took at 2048 features and 80000 rows: a score 529 against 570 us at
// 128 tokens (float32; bfloat16 236 against 253), a score and its gradients 788
// against 1240 us at 64 (float32), 445 against 620 at 32 but 870 against 628 at 64
// (bfloat16, whose backward here is on the float32 instructions).
constexpr int kFewScores = 128;
template <class T>
constexpr int kFewTokens = T::kBytes == 4 ? 64 : 32;
constexpr int kFewThreads = 256, kFewWaves = kFewThreads / kWave;

// Sixteen bytes of a row (four float32, eight bfloat16), zeros past its end.
template <class T>
using FewPiece = std::conditional_t<T::kBytes == 4, f32x4, b16x8>;
template <class T, bool VEC>
__device__ __forceinline__ FewPiece<T> few_piece(const void* p, int64_t i, int64_t left) {
    constexpr int kMine = 16 / T::kBytes;
    FewPiece<T> x;
    if (VEC) {  // the row's length is a multiple of the piece
        x = *reinterpret_cast<const FewPiece<T>*>(static_cast<const char*>(p) + i * T::kBytes);
        if (left <= 0) x = FewPiece<T>{};
    } else {
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const float v = T::load(p, j < left ? i + j : i);
            if constexpr (kMine == 4) x[j] = j < left ? v : 0.0f;
            else x[j] = static_cast<__bf16>(j < left ? v : 0.0f);
        }
    }
    return x;
}

// 16 MB rows of one operand (block blk of them; past the end the last again)
// against 16 NB of the other (few): lane l holds row l % 16 of both, piece l / 16
// of each run of 64 bytes. The same columns meet in both operands, so their order
// within an instruction does not matter. The loads of U runs are in flight
// together. Lane l, register r of acc[a][b]: row 16 a + 4 (l / 16) + r, few
// 16 b + l % 16. Columns k .. k1, whole times U runs but where k1 is d.
template <class T, bool VEC, int MB, int NB, int U>
__device__ __forceinline__ void few_products(const void* __restrict__ rows, int64_t nrows,
                                             int64_t blk, const void* __restrict__ few,
                                             const int64_t (&fo)[NB], int64_t d, int64_t k,
                                             int64_t k1, int lane, f32x4 (&acc)[MB][NB]) {
    constexpr int kMine = 16 / T::kBytes, kRun = 4 * kMine;
    const int quarter = lane >> 4;
    int64_t ro[MB];
#pragma unroll
    for (int a = 0; a < MB; ++a) {
        const int64_t row = (blk * MB + a) * 16 + (lane & 15);
        ro[a] = (row < nrows ? row : nrows - 1) * d + kMine * quarter;
    }
#pragma unroll
    for (int a = 0; a < MB; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    FewPiece<T> x[U][MB], y[U][NB];
    auto runs = [&](int64_t k, auto end) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // past the row's end: its first piece, as zeros
            const int64_t left =
                decltype(end)::value ? d - k - u * kRun - kMine * quarter : kMine;
            const int64_t at = left > 0 ? k + u * kRun : -kMine * quarter;
#pragma unroll
            for (int a = 0; a < MB; ++a) x[u][a] = few_piece<T, VEC>(rows, ro[a] + at, left);
#pragma unroll
            for (int b = 0; b < NB; ++b) y[u][b] = few_piece<T, VEC>(few, fo[b] + at, left);
        }
        __builtin_amdgcn_sched_barrier(0);  // all loads before the first product's wait
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < MB; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if constexpr (kMine == 4) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                x[u][a][j], y[u][b][j], acc[a][b], 0, 0, 0);
                    } else {
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u][a], y[u][b],
                                                                            acc[a][b], 0, 0, 0);
                    }
                }
    };
    for (; k + U * kRun <= k1; k += U * kRun) runs(k, std::false_type{});
    if (k < k1) runs(k, std::true_type{});
}

// The same with the columns split among a workgroup's four waves: z[a][b] is the
// joined sum of row 16 a + 4 (l / 16) + wv, few 16 b + l % 16.
template <class T, bool VEC, int MB, int NB, int U>
__device__ __forceinline__ void few_split(const void* __restrict__ rows, int64_t nrows,
                                          int64_t blk, const void* __restrict__ few,
                                          const int64_t (&fo)[NB], int64_t d, int wv, int lane,
                                          float (&sh)[kFewWaves][MB][NB][4][kWave],
                                          float (&z)[MB][NB]) {
    constexpr int kStep = U * 64 / T::kBytes;
    const int64_t steps = ceil_div(d, kStep);
    const int64_t k0 = steps * wv / kFewWaves * kStep, k1 = steps * (wv + 1) / kFewWaves * kStep;
    f32x4 acc[MB][NB];
    few_products<T, VEC, MB, NB, U>(rows, nrows, blk, few, fo, d, k0, k1 < d ? k1 : d, lane, acc);
    __syncthreads();  // the last block's sums are read
#pragma unroll
    for (int a = 0; a < MB; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) sh[wv][a][b][r][lane] = acc[a][b][r];
    __syncthreads();
#pragma unroll
    for (int a = 0; a < MB; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            z[a][b] = 0.0f;
#pragma unroll
            for (int k = 0; k < kFewWaves; ++k) z[a][b] += sh[k][a][b][wv][lane];
        }
}

// Forward of few tokens: a wave (SPLIT: a workgroup) takes 16 MB rows of W at a
// time against all live tokens (list[0 .. live); the last is repeated). z is kept
// for the backward where it is wanted, `pitch` tokens a row. More rows of W at a
// time read the tokens from the L2 less often; split, there are still workgroups
// enough: 64 tokens, 2048 features, 80000 rows in 317 us at 32 rows a wave, 258 at
// 64 a workgroup. 128 tokens' sums are too many for that (768 features, 32768
// rows: 76 us, split 95).
template <class T, bool VEC, int MB, int NB, int U, bool SPLIT>
__device__ __forceinline__ void few_forward(
    const void* __restrict__ h, const void* __restrict__ w, const int64_t* __restrict__ target,
    const int* list, int live, int64_t n, int64_t d, int64_t v, float2* __restrict__ part,
    float* __restrict__ zt, float* __restrict__ keep, int pitch) {
    constexpr int kMine = 16 / T::kBytes;
    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quarter = lane >> 4;
    int64_t want[NB], ho[NB];
    int tok[NB];
    float m[NB], s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const bool in = 16 * b + col < live;
        tok[b] = list[in ? 16 * b + col : live - 1];
        want[b] = in ? target[tok[b]] : -1;
        ho[b] = tok[b] * d + kMine * quarter;
        m[b] = -INFINITY;
        s[b] = 0.0f;
    }
    constexpr int R = SPLIT ? 1 : 4;  // rows of a lane and block
    const int64_t blocks = ceil_div(v, 16 * MB);
    const int64_t per = SPLIT ? 1 : kFewWaves;
    for (int64_t blk = blockIdx.x * per + (SPLIT ? 0 : wv); blk < blocks; blk += gridDim.x * per) {
        float zs[MB][NB][R];
        if constexpr (SPLIT) {
            __shared__ float sums[kFewWaves][MB][NB][4][kWave];
            float z[MB][NB];
            few_split<T, VEC, MB, NB, U>(w, v, blk, h, ho, d, wv, lane, sums, z);
#pragma unroll
            for (int a = 0; a < MB; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b) zs[a][b][0] = z[a][b];
        } else {
            f32x4 acc[MB][NB];
            few_products<T, VEC, MB, NB, U>(w, v, blk, h, ho, d, 0, d, lane, acc);
#pragma unroll
            for (int a = 0; a < MB; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < R; ++r) zs[a][b][r] = acc[a][b][r];
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float top = m[b];
#pragma unroll
            for (int a = 0; a < MB; ++a)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int64_t vr = (blk * MB + a) * 16 + 4 * quarter + (SPLIT ? wv : r);
                    float z = zs[a][b][r];
                    if (vr == want[b]) zt[tok[b]] = z;
                    if (keep != nullptr && vr < v) keep[vr * pitch + tok[b]] = z;
                    if (vr >= v) z = -INFINITY;
                    zs[a][b][r] = z;
                    top = fmaxf(top, z);
                }
            const float base = top == -INFINITY ? 0.0f : top;
            s[b] = m[b] == -INFINITY ? s[b] : s[b] * exp_(m[b] - base);
#pragma unroll
            for (int a = 0; a < MB; ++a)
#pragma unroll
                for (int r = 0; r < R; ++r) s[b] += exp_(zs[a][b][r] - base);
            m[b] = top;
        }
    }
    // the lanes of a token, then the waves
    __shared__ float2 sh[kFewWaves][16 * NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[b], o), s2 = __shfl_xor(s[b], o);
            join(m[b], s[b], m2, s2);
        }
        if (lane < 16) sh[wv][16 * b + lane] = make_float2(m[b], s[b]);
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < live) {
        float2 x = sh[0][threadIdx.x];
        for (int k = 1; k < kFewWaves; ++k)
            join(x.x, x.y, sh[k][threadIdx.x].x, sh[k][threadIdx.x].y);
        part[static_cast<int64_t>(blockIdx.x) * n + list[threadIdx.x]] = x;
    }
}

// The live tokens first, then as many blocks of 16 as they fill, of at most MOST.
template <class T, bool VEC, int MOST>
__global__ __launch_bounds__(kFewThreads) void ce_few_kernel(
    const void* __restrict__ h, const void* __restrict__ w, const int64_t* __restrict__ target,
    int64_t n, int64_t d, int64_t v, int64_t ignore, float2* __restrict__ part,
    float* __restrict__ zt, float* __restrict__ keep) {
    __shared__ int list[16 * MOST];
    const int lane = threadIdx.x & (kWave - 1);
    int live = 0;
#pragma unroll
    for (int t0 = 0; t0 < 16 * MOST; t0 += kWave) {  // every wave counts, the first writes
        const int t = t0 + lane;
        const bool in = t < n && target[t < n ? t : 0] != ignore;
        const uint64_t mask = __ballot(in);
        if (in && threadIdx.x < kWave)
            list[live + __popcll(mask & ((uint64_t{1} << lane) - 1))] = t;
        live += __popcll(mask);
    }
    __syncthreads();
    if (live == 0) return;  // the whole grid; the joined losses are 0
    constexpr int kPitch = 16 * MOST;
#define SLK_FEW(MB, NB, U, S) \
    few_forward<T, VEC, MB, NB, U, S>(h, w, target, list, live, n, d, v, part, zt, keep, kPitch)
    if constexpr (MOST >= 8) {
        if (live > 64) return SLK_FEW(2, 8, 2, false);
    }
    if constexpr (MOST >= 4) {
        if (live > 32) return SLK_FEW(4, 4, 2, true);
    }
    if constexpr (MOST >= 2) {
        if (live > 16) return SLK_FEW(2, 2, 4, false);
    }
    SLK_FEW(1, 1, 8, false);
#undef SLK_FEW
}

// Forward of a small vocabulary, the same with the operands' parts exchanged: a
// workgroup has all logits of 16 MB tokens, so their softmax and loss too. (With a
// wave for all columns of 16 tokens 8192 x 4096 x 65 float32 took 187 us, split 97,
// with 32 tokens 64: W comes from the L2 for each of them.)
template <class T, bool VEC, int MB, int NB, int U>
__global__ __launch_bounds__(kFewThreads) void ce_small_kernel(
    const void* __restrict__ h, const void* __restrict__ w, const int64_t* __restrict__ target,
    int64_t n, int64_t d, int64_t v, int64_t ignore, float* __restrict__ losses,
    float2* __restrict__ norm, float* __restrict__ keep) {
    constexpr int kMine = 16 / T::kBytes, kVoc = 16 * NB;
    __shared__ float sums[kFewWaves][MB][NB][4][kWave];
    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quarter = lane >> 4;
    int64_t wo[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
        wo[b] = (16 * b + col < v ? 16 * b + col : v - 1) * d + kMine * quarter;
    const int64_t blocks = ceil_div(n, 16 * MB);
    for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        float zs[MB][NB];
        few_split<T, VEC, MB, NB, U>(h, n, blk, w, wo, d, wv, lane, sums, zs);
#pragma unroll
        for (int a = 0; a < MB; ++a) {
            const int64_t tok = (blk * MB + a) * 16 + 4 * quarter + wv;
            const int64_t t = tok < n ? target[tok] : ignore;
            float m = -INFINITY, s = 0.0f, zt = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float z = zs[a][b];
                if (keep != nullptr && tok < n) keep[tok * kVoc + 16 * b + col] = z;
                if (16 * b + col == t) zt = z;
                zs[a][b] = 16 * b + col < v ? z : -INFINITY;
                m = fmaxf(m, zs[a][b]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
            if (m == -INFINITY) m = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) s += exp_(zs[a][b] - m);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                s += __shfl_xor(s, o);
                zt += __shfl_xor(zt, o);
            }
            if (col != 0 || tok >= n) continue;
            const bool valid = t >= 0 && t < v;
            losses[tok] = t == ignore ? 0.0f : valid ? (m - zt) + log2f(s) * kLn2 : NAN;
            if (norm != nullptr) norm[tok] = make_float2(m, 1.0f / s);
        }
    }
}

// Backward of both. Rows are those of the long operand (W of few tokens, the
// hidden states of a small vocabulary), few those of the other; both products,
//   d rows = dl·few,   d few = dlᵀ·rows     (dl rows x few),
// of a part of the rows and 256 columns, 64 a wave, on the float32 matrix
// instructions (bfloat16 is widened). Lane l holds columns 4 (l % 16) .. + 3 of
// row l / 16 of four, sixteen bytes in float32: block i of an instruction's
// columns is the lanes' i-th, so that rows are read and written in runs of 256
// bytes. The few stay in registers, as do their sums; dl is made from the logits
// in LDS, 32 rows at a time, by all waves. An ignored token's row or place in dl
// is 0, and so is what is read of its hidden state, whatever it holds.
constexpr int kFewRows = 32;  // rows between barriers
struct FewArgs {
    const void *few, *rows;
    const int64_t* target;
    const float* z;       // rows x 16 NB
    const float2* norm;   // of the tokens
    const float* up;
    const float* live;    // small vocabulary: the tokens not ignored
    int64_t nfew, nrows, d, ignore, per;  // per: rows of a part, a multiple of kFewRows
    int reduction;
    float* sums;     // d few: parts x nfew x d, NULL: not wanted
    void* drows;     // NULL: not wanted
    float* factor;   // left for the sums, with pos (few tokens)
    int32_t* pos;
};
// What a token's column (few tokens) or row (small vocabulary) of dl takes:
// p = exp(z - m)·gs, less g at hit. gs = g / s; hit -1: none, -2: ignored.
struct FewToken {
    float m, gs, g;
    int hit;
};
template <class T, bool VEC, int NB, bool SMALL>
__global__ __launch_bounds__(kFewThreads) void ce_few_back_kernel(const FewArgs p) {
    constexpr int kFew = 16 * NB, kPitch = kFew + 1, kSub = kFewRows / 16;
    constexpr int kEach = kFewRows * kFew / kFewThreads;
    __shared__ float dl[2][kFewRows * kPitch];
    __shared__ FewToken tokens[SMALL ? 3 * kFewRows : kFew];  // (SMALL: of three rounds)
    __shared__ float top_factor;
    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t r_0 = blockIdx.y * p.per;
    const int64_t r_1 = r_0 + p.per < p.nrows ? r_0 + p.per : p.nrows;
    const int64_t classes = SMALL ? p.nfew : p.nrows;

    auto token = [&](int64_t i, bool live, int64_t t, float g) {
        const float2 x = live ? p.norm[i] : make_float2(0.0f, 0.0f);
        return FewToken{x.x, live ? g * x.y : 0.0f, live ? g : 0.0f,
                        !live ? -2 : t >= 0 && t < classes ? static_cast<int>(t) : -1};
    };
    // SMALL: row r0 + threadIdx.x of the next round, of the first 32 threads
    auto row_token = [&](int64_t r0) {
        const int64_t i = r0 + threadIdx.x;
        const bool in = threadIdx.x < kFewRows && i < r_1;
        const int64_t t = in ? p.target[i] : p.ignore;
        const bool live = t != p.ignore;
        return token(i, live, t, live && p.reduction == SLK_REDUCE_NONE ? p.up[i] : 1.0f);
    };
    if constexpr (SMALL) {
        if (threadIdx.x < kFewRows) tokens[threadIdx.x] = row_token(r_0);
        if (threadIdx.x == 0) {
            float f = 1.0f;
            if (p.reduction == SLK_REDUCE_SUM) f = *p.up;
            if (p.reduction == SLK_REDUCE_MEAN) f = *p.live > 0.0f ? *p.up / *p.live : 0.0f;
            top_factor = f;
            if (blockIdx.x == 0 && blockIdx.y == 0) *p.factor = f;
        }
    } else if (wv == 0) {
        const bool in = lane < p.nfew;
        const int64_t t = in ? p.target[lane] : p.ignore;
        const bool live = in && t != p.ignore;
        const int count = __popcll(__ballot(live));
        float g = 1.0f, f = 1.0f;
        if (p.reduction == SLK_REDUCE_NONE) g = live ? p.up[lane] : 0.0f;
        else f = count == 0 ? 0.0f : p.reduction == SLK_REDUCE_MEAN ? *p.up / count : *p.up;
        if (lane < kFew) tokens[lane] = token(lane, live, t, g);
        if (lane == 0) top_factor = f;
        if (blockIdx.x == 0 && blockIdx.y == 0) {
            if (in) p.pos[lane] = live ? lane : -1;
            if (lane == 0) *p.factor = f;
        }
    }
    __syncthreads();
    const float factor = top_factor;

    const int col = lane & 15, quarter = lane >> 4;
    const int64_t c0 = blockIdx.x * 256 + 64 * wv + 4 * col;
    auto load = [&](const void* from, int64_t row, f32x4& x) {
        x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (VEC) {
            if (c0 < p.d) {
                float y[4];
                T::load4(from, row * p.d + c0, y);
                x = f32x4{y[0], y[1], y[2], y[3]};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + i < p.d) x[i] = T::load(from, row * p.d + c0 + i);
        }
    };
    f32x4 few[4 * NB];  // row 4 j + l / 16
#pragma unroll
    for (int j = 0; j < 4 * NB; ++j) {
        const int i = 4 * j + quarter;
        few[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (p.drows != nullptr && i < p.nfew && (SMALL || tokens[SMALL ? 0 : i].hit != -2))
            load(p.few, i, few[j]);
    }
    f32x4 sum[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[b][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    f32x4 x[kSub][4];  // row 16 k + 4 j + l / 16
    float zs[kEach];
    auto logits = [&](int64_t r0) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int at = k * kFewThreads + threadIdx.x;
            zs[k] = r0 + at / kFew < r_1 ? p.z[r0 * kFew + at] : 0.0f;
        }
    };
    logits(r_0);
    // dl of two rounds, tokens of three: a round's tokens are read until the next
    // round's barrier, when those of the round after are written
    int buf = 0, turn = 0;
    for (int64_t r0 = r_0; r0 < r_1; r0 += kFewRows, buf ^= 1) {
        const FewToken* mine_tokens = tokens + (SMALL ? turn * kFewRows : 0);
        turn = turn == 2 ? 0 : turn + 1;
        if (p.sums != nullptr) {
#pragma unroll
            for (int k = 0; k < kSub; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = 16 * k + 4 * j + quarter;
                    load(p.rows, r0 + i < r_1 ? r0 + i : r_1 - 1, x[k][j]);
                    if (SMALL && mine_tokens[i].hit == -2) x[k][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int at = k * kFewThreads + threadIdx.x, row = at / kFew, i = at % kFew;
            const FewToken t = mine_tokens[SMALL ? row : i];
            float g = exp_(zs[k] - t.m) * t.gs;
            if ((SMALL ? i : r0 + row) == t.hit) g -= t.g;
            dl[buf][row * kPitch + i] = r0 + row < r_1 && i < p.nfew && t.hit != -2 ? g : 0.0f;
        }
        if (r0 + kFewRows < r_1) {
            logits(r0 + kFewRows);
            if (SMALL && threadIdx.x < kFewRows)
                tokens[SMALL ? turn * kFewRows + threadIdx.x : 0] = row_token(r0 + kFewRows);
        }
        __syncthreads();  // (this dl was last read two rounds ago, a barrier ago)
        if (c0 - 4 * col >= p.d) continue;  // the whole wave: no column of its own
#pragma unroll
        for (int k = 0; k < kSub; ++k) {
            const float* mine = dl[buf] + 16 * k * kPitch;
            if (p.drows != nullptr) {
                f32x4 acc[4] = {};
#pragma unroll
                for (int j = 0; j < 4 * NB; ++j) {
                    const float a = mine[col * kPitch + 4 * j + quarter];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, few[j][i], acc[i], 0, 0,
                                                                      0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = 16 * k + 4 * quarter + r;
                    const int64_t row = r0 + at;
                    if (row >= r_1) continue;
                    const bool none = SMALL && mine_tokens[at].hit == -2;
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = none ? 0.0f : acc[i][r] * factor;
                    if (VEC) {
                        if (c0 < p.d) T::store4(p.drows, row * p.d + c0, y);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (c0 + i < p.d) T::store(p.drows, row * p.d + c0 + i, y[i]);
                    }
                }
            }
            if (p.sums != nullptr) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = mine[(4 * j + quarter) * kPitch + 16 * b + col];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sum[b][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, x[k][j][i],
                                                                             sum[b][i], 0, 0, 0);
                    }
            }
        }
    }
    if (p.sums == nullptr) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t i = 16 * b + 4 * quarter + r;
            if (i >= p.nfew) continue;
            float* to = p.sums + (blockIdx.y * p.nfew + i) * p.d + c0;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c0 + c < p.d) to[c] = sum[b][c][r];
        }
}

// ───────────────────────────── sizes ─────────────────────────────

int64_t up64(int64_t x) { return (x + 63) & ~int64_t{63}; }
int64_t up256(int64_t x) { return (x + 255) & ~int64_t{255}; }

int64_t tiled(int64_t rows) { return ceil_div(rows, kTileM) * kTileM; }

struct Carve {
    int64_t at = 0;
    int64_t take(int64_t bytes) {
        const int64_t o = at;
        at = up256(at + bytes);
        return o;
    }
};

struct Saved {
    int64_t header, rows, pos, tgt, norm, hx, wx, h, w, z, live, bytes;
};

bool split_of(const slk_linear_ce* a) { return a->dtype == SLK_F32; }
int64_t stages(const slk_linear_ce* a, int64_t k) { return ceil_div(k, split_of(a) ? 32 : 64); }

bool few(const slk_linear_ce* a) {
    return a->n <= (!a->keep ? kFewScores : split_of(a) ? kFewTokens<F32> : kFewTokens<BF16>);
}
// A small vocabulary takes the few tokens' way with the operands exchanged: the
// tiles' 256 rows of vocabulary would stay mostly empty. 8192 x 384 x 65 float32,
// forward and backward: 57 us of kernels against 107; 8192 x 4096 x 65: 261 against
// 439. Of bfloat16, whose backward is on the float32 instructions here, only up to
// 2^23 hidden values: 8192 x 1024 x 128 takes 121 us against 148, but 8192 x 4096 x
// 65 240 against 209 and 65536 x 384 x 65 255 against 198 (scores alone: 46 against
// 91, 61 against 96).
constexpr int kSmallVoc = 128;
constexpr int64_t kSmallHidden = int64_t{1} << 23;
bool small(const slk_linear_ce* a) {
    return !few(a) && a->v <= kSmallVoc &&
           (!a->keep || split_of(a) || a->n * a->d <= kSmallHidden);
}
// blocks of 16 of the few: tokens 1, 2, 4 or 8, a small vocabulary 5 or 8
int64_t few_blocks(const slk_linear_ce* a) {
    if (small(a)) return a->v <= 80 ? 5 : 8;
    return a->n <= 16 ? 1 : a->n <= 32 ? 2 : a->n <= 64 ? 4 : 8;
}

Saved saved_of(const slk_linear_ce* a) {
    Saved s{};
    Carve c;
    if (few(a) || small(a)) {  // the logits themselves
        s.norm = c.take(8 * a->n);
        s.z = c.take((small(a) ? a->n : a->v) * few_blocks(a) * 64);
        s.live = c.take(4);
        s.bytes = a->keep ? c.at : 0;
        return s;
    }
    s.header = c.take(sizeof(Header));
    s.rows = c.take(4 * a->n);
    s.pos = c.take(4 * a->n);
    s.tgt = c.take(4 * a->n);
    s.norm = c.take(8 * a->n);
    s.hx = c.take(split_of(a) ? 4 * a->n : 0);
    s.wx = c.take(split_of(a) ? 4 * tiled(a->v) : 0);
    s.h = c.take(stages(a, a->d) * up64(a->n) * kStageBytes);
    s.w = c.take(stages(a, a->d) * up64(a->v) * kStageBytes);
    s.bytes = c.at;
    return s;
}

constexpr int64_t kFewGroups = 2048;  // workgroups of ce_few_kernel at most

int64_t parts_of(const slk_linear_ce* a) {
    if (small(a)) return 0;
    if (few(a)) {
        // (the rows that ce_few_kernel's variants take at a time)
        const int64_t b = few_blocks(a);
        const int64_t g = ceil_div(a->v, b == 1 ? 16 * kFewWaves : b == 4 ? 64 : 32 * kFewWaves);
        return g < kFewGroups ? g : kFewGroups;
    }
    return ceil_div(a->v, kTileM);
}

struct Forward {
    int64_t part, zt, losses, bytes;
};
Forward forward_of(const slk_linear_ce* a) {
    Forward f;
    Carve c;
    f.part = c.take(8 * parts_of(a) * a->n);
    f.zt = c.take(4 * a->n);
    f.losses = c.take(4 * a->n);
    f.bytes = c.at;
    return f;
}

// Vocabulary rows of a piece of the backward: dl of a piece takes at most
// kDlBytes, or 256 rows over all tokens where those take more (from 2^19 tokens in
// float32, 2^20 in bfloat16), and as much again in float32 as dh's operand.
constexpr int64_t kDlBytes = int64_t{1} << 29;

// Parts of a product's K loop. With one workgroup a CU, tiles·s of them take
// ceil(tiles·s / 256) rounds of 1/s of the loop each (about 1.1 us a stage of a
// 256 x 128 tile); more than one part also writes and reads its sums.
int splits_for(int64_t m, int64_t n, int64_t nst) {
    const double sums = 1e-6 * static_cast<double>(m) * static_cast<double>(n) / 4.5;  // us a byte
    int best = 1;
    double cost = 1e30;
    for (int s = 1; s <= 32; ++s) {
        if (s > 1 && nst < 8 * s) break;
        const bool wide = mma_wide(m, n, s);
        const int64_t tiles = ceil_div(m, kTileM) * ceil_div(n, wide ? kWideN : kTileN);
        const double c = static_cast<double>(ceil_div(tiles * s, 256)) * (wide ? 1.7 : 1.0) * 1.1 *
                             static_cast<double>(nst) / s +
                         (s > 1 ? sums * (8.0 * s + 4.0) + 5.0 : 0.0);
        if (c < cost) {
            cost = c;
            best = s;
        }
    }
    return best;
}

struct Backward {
    int64_t piece;  // rows of a piece, a multiple of kTileM
    int sh, sw;     // parts of the two products
    int64_t gr, factor, pos, dl, dlh, dl_rows, dh, dw, bytes;
    int64_t row_part, col_part, row_exp, col_exp;  // float32
};
Backward backward_of(const slk_linear_ce* a) {
    Backward b{};
    if (few(a) || small(a)) {
        // parts of the rows: two workgroups a CU over all columns, or (a small
        // vocabulary: few rows a part and all its sums to join, or registers for
        // one) one
        const int64_t nrows = small(a) ? a->n : a->v, nfew = small(a) ? a->v : a->n;
        const int64_t cols = ceil_div(a->d, 256);
        const bool one = small(a) && (few_blocks(a) == 8 || nrows * cols < 512 * 128);
        const int64_t most = ceil_div(one ? 256 : 512, cols);
        b.piece = ceil_div(ceil_div(nrows, most), kFewRows) * kFewRows;
        b.sh = static_cast<int>(ceil_div(nrows, b.piece));
        Carve c;
        b.factor = c.take(4);
        b.pos = c.take(small(a) ? 0 : 4 * a->n);
        b.dh = c.take((small(a) ? a->dweight : a->dhidden) != nullptr ? 4 * b.sh * nfew * a->d : 0);
        b.bytes = c.at;
        return b;
    }
    // (the epilogue writes whole tiles of tokens)
    b.dl_rows = ceil_div(a->n, kWideN) * kWideN;
    const int64_t per_row = b.dl_rows * (split_of(a) ? 4 : 2);
    int64_t most = kDlBytes / per_row / kTileM * kTileM;  // rows of a piece
    if (most < kTileM) most = kTileM;
    const int64_t all = ceil_div(a->v, kTileM) * kTileM;
    if (most > all) most = all;
    // as few pieces as fit, or a few more where their tiles fill the last round of
    // the 256 CUs better: stages of a tile times rounds, and dh read and written
    // once a piece (about 130 stages' time at 8192 x 4096)
    double cost = 1e30;
    for (int64_t k = ceil_div(all, most); k < ceil_div(all, most) + 4; ++k) {
        const int64_t rows = ceil_div(ceil_div(all, k), kTileM) * kTileM;
        double c = 0.0;
        for (int64_t v0 = 0; v0 < a->v; v0 += rows) {
            const int64_t vn = a->v - v0 < rows ? a->v - v0 : rows;
            c += mma_rounds(vn, a->n) * static_cast<double>(stages(a, a->d)) +
                 mma_rounds(vn, a->d) * static_cast<double>(stages(a, a->n)) +
                 mma_rounds(a->n, a->d) * static_cast<double>(stages(a, vn)) + 20.0 +
                 static_cast<double>(a->n) * static_cast<double>(a->d) * 4e-6;
        }
        if (c < cost) {
            cost = c;
            b.piece = rows;
        }
    }
    b.sh = splits_for(a->n, a->d, stages(a, b.piece));
    b.sw = splits_for(b.piece, a->d, stages(a, a->n));
    Carve c;
    b.factor = c.take(4);
    b.gr = c.take(4 * a->n);
    b.dl = c.take(stages(a, b.piece) * b.dl_rows * kStageBytes);
    if (split_of(a)) {
        b.dlh = c.take(a->dhidden != nullptr ? stages(a, b.piece) * b.dl_rows * kStageBytes : 0);
        b.row_part = c.take(4 * b.piece / kTileM * b.dl_rows);
        b.col_part = c.take(4 * b.dl_rows / kTileN * b.piece);
        b.row_exp = c.take(4 * b.dl_rows);
        b.col_exp = c.take(4 * b.piece);
    }
    const bool whole = b.sh == 1 && b.piece >= a->v;
    b.dh = c.take(a->dhidden != nullptr && !whole ? 4 * b.sh * a->n * a->d : 0);
    b.dw = c.take(a->dweight != nullptr && b.sw > 1 ? 4 * b.sw * b.piece * a->d : 0);
    b.bytes = c.at;
    return b;
}

int validate(const slk_linear_ce* a, const char* who) {
    const std::string w(who);
    if (a == nullptr) return fail(SLK_EINVAL, w + ": NULL arguments");
    if (a->n < 0 || a->d < 1 || a->v < 1) {
        return fail(SLK_EINVAL, w + ": n must be >= 0, d and v >= 1");
    }
    if (a->n > (1 << 25) || a->v > (1 << 25) || a->d > (1 << 20)) {
        return fail(SLK_EINVAL, w + ": at most 2^25 tokens and vocabulary rows, 2^20 features");
    }
    if (a->dtype != SLK_F32 && a->dtype != SLK_BF16) {
        return fail(SLK_EINVAL, w + ": dtype must be SLK_F32 or SLK_BF16");
    }
    if (a->reduction != SLK_REDUCE_NONE && a->reduction != SLK_REDUCE_SUM &&
        a->reduction != SLK_REDUCE_MEAN) {
        return fail(SLK_EINVAL, w + ": unknown reduction");
    }
    if (a->n > 0 && !few(a) && !small(a) &&
        ceil_div(a->v, kTileM) * ceil_div(a->n, mma_wide(a->v, a->n, 1) ? kWideN : kTileN) >
            max_groups(kMmaThreads)) {
        return fail(SLK_EINVAL, w + ": too many logits in a call: n=" + std::to_string(a->n) +
                                    ", v=" + std::to_string(a->v));
    }
    return SLK_OK;
}

template <class T, bool SPLIT>
int pack(const PackArgs& p, hipStream_t st) {
    constexpr int K = kStageK<SPLIT>;
    const dim3 grid(static_cast<unsigned>(ceil_div(ceil_div(up64(p.R), 4) * (K / 8), 256)),
                    static_cast<unsigned>(ceil_div(p.d, K)));
    const bool vec = p.d % 4 == 0 && aligned_to(p.src, 4 * T::kBytes);
    if (vec) hipLaunchKernelGGL((ce_pack_kernel<T, SPLIT, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((ce_pack_kernel<T, SPLIT, false>), grid, dim3(256), 0, st, p);
    return check_launch("linear_ce pack");
}

template <class T, bool SPLIT>
int forward(const slk_linear_ce* a, hipStream_t st) {
    const Forward f = forward_of(a);
    char* sc = static_cast<char*>(a->scratch);
    float2* part = reinterpret_cast<float2*>(sc + f.part);
    float* zt = reinterpret_cast<float*>(sc + f.zt);
    float* losses = a->reduction == SLK_REDUCE_NONE ? a->loss
                                                    : reinterpret_cast<float*>(sc + f.losses);
    JoinArgs j{part, zt, a->target, nullptr, nullptr, nullptr, losses, a->n, a->v,
               a->ignore_index, parts_of(a)};
    int rc = SLK_OK;
    float *z = nullptr, *live = nullptr;
    if (a->keep && (few(a) || small(a))) {
        char* sv = static_cast<char*>(a->saved);
        z = reinterpret_cast<float*>(sv + saved_of(a).z);
        j.norm = reinterpret_cast<float2*>(sv + saved_of(a).norm);
        live = reinterpret_cast<float*>(sv + saved_of(a).live);
    }
    const bool vec = a->d % (16 / T::kBytes) == 0 && aligned_to(a->hidden, 16) &&
                     aligned_to(a->weight, 16);
    if (small(a)) {
        const bool more = a->n >= 8192;  // 32 tokens a workgroup, which fill the card
        const int64_t g = ceil_div(a->n, more ? 32 : 16);
        auto go = [&](auto k) {
            hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(g < 4096 ? g : 4096)),
                               dim3(kFewThreads), 0, st, a->hidden, a->weight, a->target, a->n,
                               a->d, a->v, a->ignore_index, losses, j.norm, z);
        };
        auto pick = [&](auto mb, auto nb) {
            constexpr int MB = decltype(mb)::value, NB = decltype(nb)::value;
            if (vec) go(ce_small_kernel<T, true, MB, NB, 2>);
            else go(ce_small_kernel<T, false, MB, NB, 2>);
        };
        std::integral_constant<int, 1> one{};
        std::integral_constant<int, 2> two{};
        std::integral_constant<int, 5> five{};
        std::integral_constant<int, 8> eight{};
        if (few_blocks(a) == 5) more ? pick(two, five) : pick(one, five);
        else more ? pick(two, eight) : pick(one, eight);
        rc = check_launch("linear_ce small");
    } else if (few(a)) {
        const dim3 grid(static_cast<unsigned>(parts_of(a)));
        auto go = [&](auto k) {
            hipLaunchKernelGGL(k, grid, dim3(kFewThreads), 0, st, a->hidden, a->weight, a->target,
                               a->n, a->d, a->v, a->ignore_index, part, zt, z);
        };
        auto pick = [&](auto most) {
            constexpr int MOST = decltype(most)::value;
            if (vec) go(ce_few_kernel<T, true, MOST>);
            else go(ce_few_kernel<T, false, MOST>);
        };
        switch (few_blocks(a)) {
            case 1: pick(std::integral_constant<int, 1>{}); break;
            case 2: pick(std::integral_constant<int, 2>{}); break;
            case 4: pick(std::integral_constant<int, 4>{}); break;
            default: pick(std::integral_constant<int, 8>{});
        }
        rc = check_launch("linear_ce few");
    } else {
        const Saved s = saved_of(a);
        char* sv = static_cast<char*>(a->saved);
        Header* hd = reinterpret_cast<Header*>(sv + s.header);
        int32_t* rows = reinterpret_cast<int32_t*>(sv + s.rows);
        int32_t* pos = reinterpret_cast<int32_t*>(sv + s.pos);
        int32_t* tgt = reinterpret_cast<int32_t*>(sv + s.tgt);
        int32_t* hx = reinterpret_cast<int32_t*>(sv + s.hx);
        int32_t* wx = reinterpret_cast<int32_t*>(sv + s.wx);
        hipLaunchKernelGGL(ce_list_kernel, dim3(1), dim3(kListThreads), 0, st, a->target, a->n,
                           a->v, a->ignore_index, hd, rows, pos, tgt);
        if ((rc = check_launch("linear_ce list")) != SLK_OK) return rc;
        if (SPLIT) {
            const int64_t g = ceil_div(a->n + a->v, 4);
            const dim3 grid(static_cast<unsigned>(g < 1024 ? g : 1024));
            const bool vec = a->d % 4 == 0 && aligned_to(a->hidden, 16) && aligned_to(a->weight, 16);
            auto go = [&](auto k) {
                hipLaunchKernelGGL(k, grid, dim3(256), 0, st, static_cast<const float*>(a->hidden),
                                   a->n, static_cast<const float*>(a->weight), a->v, tiled(a->v),
                                   a->d, pos, hx, wx);
            };
            if (vec) go(ce_exp_kernel<true>);
            else go(ce_exp_kernel<false>);
            if ((rc = check_launch("linear_ce scales")) != SLK_OK) return rc;
        }
        const PackArgs ph{a->hidden, rows, &hd->live, hx, a->n, a->d, up64(a->n), sv + s.h};
        const PackArgs pw{a->weight, nullptr, nullptr, wx, a->v, a->d, up64(a->v), sv + s.w};
        if ((rc = pack<T, SPLIT>(ph, st)) != SLK_OK) return rc;
        if ((rc = pack<T, SPLIT>(pw, st)) != SLK_OK) return rc;
        const MmaArgs g{sv + s.w, sv + s.h, a->v, a->n, stages(a, a->d), up64(a->v), up64(a->n),
                        &hd->live, kLiveN, 1};
        rc = mma<SPLIT, false, false>(g, ScoreEpi<SPLIT>{wx, hx, tgt, part, zt, a->n}, st,
                                      "linear_ce logits");
        j.pos = pos;
        j.tgt = tgt;
        j.norm = reinterpret_cast<float2*>(sv + s.norm);
    }
    if (rc != SLK_OK) return rc;
    if (small(a)) {
        // the losses are there
    } else if (few(a)) {
        hipLaunchKernelGGL(ce_join_kernel<1>, dim3(static_cast<unsigned>(a->n)), dim3(256), 0, st,
                           j);
    } else {
        hipLaunchKernelGGL(ce_join_kernel<8>, dim3(static_cast<unsigned>(ceil_div(a->n, 8))),
                           dim3(256), 0, st, j);
    }
    if ((rc = check_launch("linear_ce join")) != SLK_OK) return rc;
    if (a->reduction != SLK_REDUCE_NONE) {
        hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(1024), 0, st, losses, a->target, a->n,
                           a->ignore_index, a->reduction == SLK_REDUCE_MEAN, live, a->loss);
        rc = check_launch("linear_ce reduce");
    }
    return rc;
}

template <class T>
int backward_few(const slk_linear_ce* a, hipStream_t st) {
    const Saved s = saved_of(a);
    const Backward b = backward_of(a);
    const char* sv = static_cast<const char*>(a->saved);
    char* sc = static_cast<char*>(a->scratch);
    const bool sm = small(a);
    void* few_out = sm ? a->dweight : a->dhidden;
    void* rows_out = sm ? a->dhidden : a->dweight;
    if (few_out == nullptr && rows_out == nullptr) return SLK_OK;
    float* sums = few_out != nullptr ? reinterpret_cast<float*>(sc + b.dh) : nullptr;
    float* factor = reinterpret_cast<float*>(sc + b.factor);
    int32_t* pos = sm ? nullptr : reinterpret_cast<int32_t*>(sc + b.pos);
    const int64_t nfew = sm ? a->v : a->n, nrows = sm ? a->n : a->v;
    const FewArgs p{sm ? a->weight : a->hidden, sm ? a->hidden : a->weight, a->target,
                    reinterpret_cast<const float*>(sv + s.z),
                    reinterpret_cast<const float2*>(sv + s.norm), a->upstream,
                    reinterpret_cast<const float*>(sv + s.live), nfew, nrows, a->d,
                    a->ignore_index, b.piece, a->reduction, sums, rows_out, factor, pos};
    const dim3 grid(static_cast<unsigned>(ceil_div(a->d, 256)), static_cast<unsigned>(b.sh));
    const bool vec = a->d % 4 == 0 && aligned_to(a->hidden, 4 * T::kBytes) &&
                     aligned_to(a->weight, 4 * T::kBytes) &&
                     aligned_to(rows_out, 4 * T::kBytes);
    auto go = [&](auto blocks, auto swapped) {
        constexpr int NB = decltype(blocks)::value;
        constexpr bool SMALL = decltype(swapped)::value;
        if (vec)
            hipLaunchKernelGGL((ce_few_back_kernel<T, true, NB, SMALL>), grid, dim3(kFewThreads),
                               0, st, p);
        else
            hipLaunchKernelGGL((ce_few_back_kernel<T, false, NB, SMALL>), grid, dim3(kFewThreads),
                               0, st, p);
    };
    using std::false_type;
    using std::true_type;
    if (sm && few_blocks(a) == 5) go(std::integral_constant<int, 5>{}, true_type{});
    else if (sm) go(std::integral_constant<int, 8>{}, true_type{});
    else if (few_blocks(a) == 1) go(std::integral_constant<int, 1>{}, false_type{});
    else if (few_blocks(a) == 2) go(std::integral_constant<int, 2>{}, false_type{});
    else if constexpr (kFewTokens<T> > 32) go(std::integral_constant<int, 4>{}, false_type{});
    int rc = check_launch("linear_ce few backward");
    if (rc != SLK_OK || sums == nullptr) return rc;
    const int64_t g = ceil_div(nfew * a->d, 256);
    hipLaunchKernelGGL(ce_finish_kernel<T>, dim3(static_cast<unsigned>(g < 8192 ? g : 8192)),
                       dim3(256), 0, st, sums, b.sh, nfew, nfew, a->d, pos, factor, nullptr,
                       few_out);
    return check_launch("linear_ce finish");
}

template <class T, bool SPLIT>
int backward(const slk_linear_ce* a, hipStream_t st) {
    if (few(a) || small(a)) return backward_few<T>(a, st);
    const Saved s = saved_of(a);
    const Backward b = backward_of(a);
    char* sv = static_cast<char*>(a->saved);
    char* sc = static_cast<char*>(a->scratch);
    const Header* hd = reinterpret_cast<const Header*>(sv + s.header);
    const int32_t* rows = reinterpret_cast<const int32_t*>(sv + s.rows);
    const int32_t* pos = reinterpret_cast<const int32_t*>(sv + s.pos);
    const int32_t* tgt = reinterpret_cast<const int32_t*>(sv + s.tgt);
    const float2* norm = reinterpret_cast<const float2*>(sv + s.norm);
    float* factor = reinterpret_cast<float*>(sc + b.factor);
    float* gr = reinterpret_cast<float*>(sc + b.gr);
    const bool whole = b.sh == 1 && b.piece >= a->v;  // a tile of dh has its whole sum
    const int64_t clears = whole && a->dhidden != nullptr ? ceil_div(a->n, 1024) : 0;
    hipLaunchKernelGGL(ce_upstream_kernel<T>,
                       dim3(static_cast<unsigned>(1 + (clears < 256 ? clears : 256))), dim3(1024),
                       0, st, a->upstream, hd, rows, a->reduction, gr, factor, pos, a->n, a->d,
                       a->dhidden);
    int rc = check_launch("linear_ce upstream");
    if (rc != SLK_OK) return rc;
    float* dh = reinterpret_cast<float*>(sc + b.dh);
    float* dw = reinterpret_cast<float*>(sc + b.dw);
    auto finish = [&](const float* sums, int splits, int64_t r, int64_t stride,
                      const int32_t* ps, const float* each, void* out) {
        const int64_t g = ceil_div(r * a->d, 256);
        hipLaunchKernelGGL(ce_finish_kernel<T>, dim3(static_cast<unsigned>(g < 8192 ? g : 8192)),
                           dim3(256), 0, st, sums, splits, r, stride, a->d, ps, factor, each, out);
        return check_launch("linear_ce finish");
    };
    const float* each = a->reduction == SLK_REDUCE_NONE ? gr : nullptr;
    // bfloat16: dl holds each token's upstream gradient already
    const float* each_h = SPLIT ? each : nullptr;
    auto ints = [&](int64_t at) { return reinterpret_cast<int32_t*>(sc + at); };
    int32_t* row_exp = SPLIT ? ints(b.row_exp) : nullptr;
    int32_t* col_exp = SPLIT ? ints(b.col_exp) : nullptr;
    char* dlh = SPLIT ? sc + b.dlh : sc + b.dl;  // dh's operand
    // The tiles of the forward's logits, whatever the piece: logits summed in another
    // order differ in their last bit, which is 6% of a softmax entry at 1e6.
    const bool wide = mma_wide(a->v, a->n, 1);
    for (int64_t v0 = 0; v0 < a->v; v0 += b.piece) {
        const int64_t vn = a->v - v0 < b.piece ? a->v - v0 : b.piece;
        const MmaArgs gl{sv + s.w + v0 * kStageBytes, sv + s.h, vn, a->n, stages(a, a->d),
                         up64(a->v), up64(a->n), &hd->live, kLiveN, 1};
        if constexpr (SPLIT) {
            const int32_t* hx = reinterpret_cast<const int32_t*>(sv + s.hx);
            const int32_t* wx = reinterpret_cast<const int32_t*>(sv + s.wx) + v0;
            const DlEpi<true> el{wx, hx, tgt, norm, each, sc + b.dl, v0, b.dl_rows,
                                 ints(b.row_part), ints(b.col_part), b.piece};
            rc = mma<true, false, false>(gl, el, st, "linear_ce dlogits", wide);
            if (rc != SLK_OK) return rc;
            const TermArgs ta{ints(b.row_part), ints(b.col_part), &hd->live, b.dl_rows, b.piece, vn,
                              wide ? kWideN : kTileN, row_exp, col_exp};
            hipLaunchKernelGGL(ce_term_kernel,
                               dim3(static_cast<unsigned>((b.dl_rows + b.piece) / 32)), dim3(256),
                               0, st, ta);
            if ((rc = check_launch("linear_ce terms")) != SLK_OK) return rc;
            const DlArgs da{sc + b.dl, a->dhidden != nullptr ? dlh : nullptr,
                            a->dweight != nullptr, wx, hx, row_exp, col_exp, each, &hd->live,
                            b.dl_rows};
            hipLaunchKernelGGL(ce_split_kernel,
                               dim3(static_cast<unsigned>(ceil_div(up64(a->n), 256)),
                                    static_cast<unsigned>(stages(a, vn))),
                               dim3(256), 0, st, da);
            if ((rc = check_launch("linear_ce split")) != SLK_OK) return rc;
        } else {
            const DlEpi<false> el{tgt, norm, each, sc + b.dl, v0, b.dl_rows};
            rc = mma<false, false, false>(gl, el, st, "linear_ce dlogits", wide);
            if (rc != SLK_OK) return rc;
        }
        if (a->dhidden != nullptr) {
            // dh = dl·W: W's rows, from v0, run along K
            const MmaArgs g{dlh, sv + s.w + v0 * kStageBytes, a->n, a->d, stages(a, vn),
                            b.dl_rows, up64(a->v), &hd->live, kLiveM, b.sh};
            if (whole) {
                rc = mma<SPLIT, false, true>(
                    g, TokenEpi<T, SPLIT>{row_exp, factor, each_h, rows, a->dhidden, a->d}, st,
                    "linear_ce dhidden");
            } else {
                rc = mma<SPLIT, false, true>(g, SumEpi<SPLIT>{dh, row_exp, a->n, a->d, v0 > 0}, st,
                                             "linear_ce dhidden");
            }
            if (rc != SLK_OK) return rc;
        }
        if (a->dweight != nullptr) {
            // dW = dlᵀ·h: both operands' rows, the tokens, run along K
            const MmaArgs g{sc + b.dl, sv + s.h, vn, a->d, stages(a, a->n), b.dl_rows,
                            up64(a->n), &hd->live, kLiveK, b.sw};
            void* out = static_cast<char*>(a->dweight) + v0 * a->d * T::kBytes;
            if (b.sw == 1) {
                rc = mma<SPLIT, true, true>(g, WeightEpi<T, SPLIT>{col_exp, factor, out, a->d}, st,
                                            "linear_ce dweight");
            } else {
                rc = mma<SPLIT, true, true>(g, SumEpi<SPLIT>{dw, col_exp, b.piece, a->d, false}, st,
                                            "linear_ce dweight");
                if (rc == SLK_OK) rc = finish(dw, b.sw, vn, b.piece, nullptr, nullptr, out);
            }
            if (rc != SLK_OK) return rc;
        }
    }
    if (a->dhidden != nullptr && !whole) rc = finish(dh, b.sh, a->n, a->n, pos, each_h, a->dhidden);
    return rc;
}

}  // namespace
}  // namespace slk

extern "C" int64_t slk_linear_ce_saved_bytes(const slk_linear_ce* a) {
    using namespace slk;
    return validate(a, "linear_ce_saved_bytes") == SLK_OK && a->n > 0 ? saved_of(a).bytes : 0;
}

extern "C" int64_t slk_linear_ce_scratch_bytes(const slk_linear_ce* a, int backward) {
    using namespace slk;
    if (validate(a, "linear_ce_scratch_bytes") != SLK_OK || a->n == 0) return 0;
    return backward ? backward_of(a).bytes : forward_of(a).bytes;
}

extern "C" int slk_linear_ce_forward(const slk_linear_ce* a, void* stream) {
    using namespace slk;
    clear_error();
    const int rc = validate(a, "linear_ce_forward");
    if (rc != SLK_OK || a->n == 0) return rc;
    if (a->hidden == nullptr || a->weight == nullptr || a->target == nullptr ||
        a->loss == nullptr) {
        return fail(SLK_EINVAL, "linear_ce_forward: NULL hidden, weight, target or loss");
    }
    if (a->scratch_bytes < forward_of(a).bytes || a->saved_bytes < saved_of(a).bytes ||
        a->scratch == nullptr || (a->saved == nullptr && saved_of(a).bytes > 0)) {
        return fail(SLK_EINVAL, "linear_ce_forward: saved or scratch too small");
    }
    if (!aligned_to(a->saved, 16) || !aligned_to(a->scratch, 16)) {
        return fail(SLK_EINVAL, "linear_ce_forward: saved and scratch must be 16-byte aligned");
    }
    return a->dtype == SLK_F32 ? forward<F32, true>(a, as_stream(stream))
                               : forward<BF16, false>(a, as_stream(stream));
}

extern "C" int slk_linear_ce_backward(const slk_linear_ce* a, void* stream) {
    using namespace slk;
    clear_error();
    const int rc = validate(a, "linear_ce_backward");
    if (rc != SLK_OK || a->n == 0) return rc;
    if (!a->keep) return fail(SLK_EINVAL, "linear_ce_backward: the forward kept nothing");
    if (a->upstream == nullptr) return fail(SLK_EINVAL, "linear_ce_backward: NULL upstream");
    if (a->scratch_bytes < backward_of(a).bytes || a->saved_bytes < saved_of(a).bytes ||
        a->scratch == nullptr || a->saved == nullptr) {
        return fail(SLK_EINVAL, "linear_ce_backward: saved or scratch too small");
    }
    if (!aligned_to(a->saved, 16) || !aligned_to(a->scratch, 16)) {
        return fail(SLK_EINVAL, "linear_ce_backward: saved and scratch must be 16-byte aligned");
    }
    if ((few(a) || small(a)) &&
        (a->hidden == nullptr || a->weight == nullptr || a->target == nullptr)) {
        return fail(SLK_EINVAL, "linear_ce_backward: NULL hidden, weight or target");
    }
    return a->dtype == SLK_F32 ? backward<F32, true>(a, as_stream(stream))
                               : backward<BF16, false>(a, as_stream(stream));
}
