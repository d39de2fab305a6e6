// Backward of the residual norm, slk_norm_backward. With xhat and rstd of pre,
// uhat and prstd of post, a = dy ∘ weight:
//   g    = dr + rstd·(a - mean(a) - xhat·mean(a ∘ xhat))        (RMSNorm: no mean(a))
//   dx   = g            do = scale·g         dgate = do ∘ post(u), summed over its tokens
//   dweight = Σ dy ∘ xhat,  dbias = Σ dy     (over tokens)
//   b    = do ∘ gate,   dpost_weight = Σ b ∘ uhat,  dpost_bias = Σ b
//   du   = prstd·(a' - mean(a') - uhat·mean(a' ∘ uhat)),  a' = b ∘ post_weight
// xhat comes from r as it was stored: rounded in bfloat16, where a second, unrounded copy
// would cost the forward and this pass 4 bytes a feature each.
// One pass over the arrays (24 bytes a feature in float32 without a gate),
// bound by memory. The sums over tokens stay in each lane's registers over the
// consecutive tokens of its team and are then written as partial rows, which a
// second kernel adds in a fixed order: no atomics, so results repeat. 16384 x 4096
// bfloat16 with both norms and a gate 178 us under the profiler, 8192 x 384 float32
// feature-major 15.8, the second kernel 4 to 5.
#include "norm.hpp"

namespace slk {
namespace {

// The sums over all tokens, as rows of a partial: dweight, dbias,
// dpost_weight, dpost_bias, and dgate where one gate serves all tokens.
constexpr int kColSums = 5;

struct BwdRow {
    const void *r, *gate, *weight, *post_weight, *post_bias;
    const void *dr, *dy, *branch;
    void *dx, *dbranch, *dgate;
    const float* stats;
    float* partial;       // workgroups x arrays x d
    float* gate_partial;  // teams x 2 x d, where a gate serves some tokens
    int64_t n, per_gate, per_team;
    int d, arrays;
    int at[kColSums];  // row of each sum in a partial, -1: not wanted
    bool layer, need_u;
    float scale, inv_d;
};

// A lane's sums: dweight, dbias, dpost_weight, dpost_bias over its team's
// tokens, and dgate (over all of them, or since the last flush).
template <int EPL>
struct Acc {
    float v[kColSums][EPL];
};
constexpr int kGateSum = 4;

// One token: dy, xh (r), g (dr) and the branch u as this lane's features; leaves
// dx in g and dbranch in u. vec(k, v) gives v the features of weight (k = 0),
// post_weight (1), post_bias (2) or the token's gate (3). POST and GATE are
// compile-time: without them their sums take no registers. Features past d hold
// 0 in every array read, so they add nothing to a sum; what they leave in g and
// u is not stored.
template <int EPL, bool POST, bool GATE, class Vec, class Sum, class Dx>
__device__ __forceinline__ void backward_row(const BwdRow& p, const f32x4 st, float (&dy)[EPL],
                                             float (&xh)[EPL], float (&g)[EPL], float (&u)[EPL],
                                             Acc<EPL>& acc, Vec&& vec, Sum& sum, Dx&& store_dx) {
    float s[EPL];
    if (p.dy != nullptr) {
        vec(0, s);
        float m[2] = {0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            xh[q] = (xh[q] - st[0]) * st[1];
            acc.v[0][q] = fmaf(dy[q], xh[q], acc.v[0][q]);
            acc.v[1][q] += dy[q];
            s[q] *= dy[q];
            m[0] += s[q];
            m[1] = fmaf(s[q], xh[q], m[1]);
        }
        sum(m);
        // g += rstd·(s - ma - xh·mx)
        const float ma = p.layer ? m[0] * p.inv_d * st[1] : 0.0f, mx = m[1] * p.inv_d * st[1];
#pragma unroll
        for (int q = 0; q < EPL; ++q)
            g[q] = fmaf(-xh[q], mx, fmaf(st[1], s[q], g[q] - ma));
    }
    store_dx(g);
    if (!p.need_u && p.dbranch == nullptr) return;
#pragma unroll
    for (int q = 0; q < EPL; ++q) g[q] *= p.scale;
    if (POST) {
#pragma unroll
        for (int q = 0; q < EPL; ++q) u[q] = (u[q] - st[2]) * st[3];  // uhat
    }
    if (GATE) {
        if (p.dgate != nullptr || p.at[kGateSum] >= 0) {
            if (POST) {
                float o[EPL];
                vec(1, o);
                if (p.post_bias != nullptr) {
                    vec(2, s);
#pragma unroll
                    for (int q = 0; q < EPL; ++q) o[q] = fmaf(u[q], o[q], s[q]);
                } else {
#pragma unroll
                    for (int q = 0; q < EPL; ++q) o[q] *= u[q];
                }
#pragma unroll
                for (int q = 0; q < EPL; ++q)
                    acc.v[kGateSum][q] = fmaf(g[q], o[q], acc.v[kGateSum][q]);
            } else {
#pragma unroll
                for (int q = 0; q < EPL; ++q)
                    acc.v[kGateSum][q] = fmaf(g[q], u[q], acc.v[kGateSum][q]);
            }
        }
        vec(3, s);
#pragma unroll
        for (int q = 0; q < EPL; ++q) g[q] *= s[q];
    }
    if (POST) {
        float m[2] = {0.0f, 0.0f};
        vec(1, s);
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            acc.v[2][q] = fmaf(g[q], u[q], acc.v[2][q]);
            acc.v[3][q] += g[q];
            s[q] *= g[q];
            m[0] += s[q];
            m[1] = fmaf(s[q], u[q], m[1]);
        }
        sum(m);
        const float ma = p.layer ? m[0] * p.inv_d * st[3] : 0.0f, mx = m[1] * p.inv_d * st[3];
#pragma unroll
        for (int q = 0; q < EPL; ++q) u[q] = fmaf(-u[q], mx, fmaf(st[3], s[q], -ma));
    } else {
#pragma unroll
        for (int q = 0; q < EPL; ++q) u[q] = g[q];
    }
}

template <int EPL>
__device__ __forceinline__ void clear(float (&v)[EPL]) {
#pragma unroll
    for (int q = 0; q < EPL; ++q) v[q] = 0.0f;
}

// A partial row, float32 in the lane's own layout.
template <int EPL, int TW, bool VEC>
__device__ __forceinline__ void store_f32(float* to, int d, int l, const float (&v)[EPL]) {
    using Lay = RowLay<EPL, TW, VEC>;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = Lay::at(q, l);
        if (e < d) to[e] = v[q];
    }
}

// The tokens that share a gate's row, followed token by token (a division a
// token costs more than its arithmetic).
struct GateRun {
    int64_t row, lo, hi;  // the gate's row, its tokens [lo, hi)
    __device__ __forceinline__ GateRun(const BwdRow& p, int64_t n)
        : row(n / p.per_gate), lo(row * p.per_gate), hi(lo + p.per_gate) {}
    __device__ __forceinline__ void next(const BwdRow& p, int64_t n) {
        if (n == hi) {
            ++row;
            lo = hi;
            hi += p.per_gate;
        }
    }
};

// dgate of a run's tokens in [t0, t1), a team's: the gate's own gradient if they
// are the whole run, else a partial row: a team has at most two, of the run
// that began before it (slot 0) and of the one that goes on after it (slot 1).
template <class T, int EPL, int TW, bool VEC>
__device__ __forceinline__ void flush(const BwdRow& p, int64_t team, int64_t t0, int64_t t1,
                                      const GateRun& run, int l, float (&dgate)[EPL]) {
    if (run.lo >= t0 && run.hi <= t1)
        row_store<T, EPL, TW, VEC>(p.dgate, run.row * p.d, p.d, l, dgate);
    else
        store_f32<EPL, TW, VEC>(p.gate_partial + (2 * team + (run.lo < t0 ? 0 : 1)) * p.d, p.d, l,
                                dgate);
    clear(dgate);
}

// Adds the workgroup's teams' sums in LDS, team by team, and writes its partial
// rows. sh: TEAMS x d floats.
template <int EPL, int TW, bool VEC, int TEAMS>
__device__ __forceinline__ void write_partials(const BwdRow& p, int64_t group, int team, int l,
                                               const Acc<EPL>& acc, float* sh) {
#pragma unroll
    for (int k = 0; k < kColSums; ++k) {
        if (p.at[k] < 0) continue;  // the same for every thread
        float* to = p.partial + (group * p.arrays + p.at[k]) * p.d;
        if (TEAMS == 1) {
            store_f32<EPL, TW, VEC>(to, p.d, l, acc.v[k]);
        } else {
            store_f32<EPL, TW, VEC>(sh + team * p.d, p.d, l, acc.v[k]);
            __syncthreads();
            for (int e = threadIdx.x; e < p.d; e += TEAMS * TW * kWave) {
                float s = sh[e];
#pragma unroll
                for (int t = 1; t < TEAMS; ++t) s += sh[t * p.d + e];
                to[e] = s;
            }
            __syncthreads();
        }
    }
}

// backward_row with the vectors loaded where they are used.
template <class T, int EPL, int TW, bool VEC, bool POST, bool GATE, class Sum>
__device__ __forceinline__ void backward_token(const BwdRow& p, int64_t n, int64_t gate_row, int l,
                                               float (&dy)[EPL], float (&r)[EPL], float (&g)[EPL],
                                               float (&u)[EPL], Acc<EPL>& acc, Sum& sum) {
    const f32x4 st = *reinterpret_cast<const f32x4*>(p.stats + 4 * n);
    auto vec = [&](int k, float (&v)[EPL]) {
        const void* from = k == 0 ? p.weight : k == 1 ? p.post_weight : k == 2 ? p.post_bias
                                                                              : p.gate;
        row_load<T, EPL, TW, VEC>(from, k == 3 ? gate_row * p.d : 0, p.d, l, v);
    };
    auto store_dx = [&](const float (&v)[EPL]) {
        if (p.dx != nullptr) row_store<T, EPL, TW, VEC>(p.dx, n * p.d, p.d, l, v);
    };
    backward_row<EPL, POST, GATE>(p, st, dy, r, g, u, acc, vec, sum, store_dx);
}

template <class T, int EPL, int TW, bool VEC, bool POST, bool GATE>
__global__ __launch_bounds__(TW > 4 ? TW * kWave : kNormThreads) void norm_backward_kernel(
    const BwdRow p) {
    constexpr int kTeams = TW == 1 ? kNormThreads / kWave : 1;
    extern __shared__ float sh[];  // TW > 1: 4 TW floats; else kTeams x d
    TeamSum<TW, 2> sum{sh};
    const int l = TW == 1 ? threadIdx.x & (kWave - 1) : threadIdx.x;
    const int mine = TW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int64_t team = static_cast<int64_t>(blockIdx.x) * kTeams + mine;
    const int64_t begin = team * p.per_team;
    const int64_t end = begin + p.per_team < p.n ? begin + p.per_team : p.n;
    Acc<EPL> acc;
#pragma unroll
    for (int k = 0; k < kColSums; ++k) clear(acc.v[k]);
    GateRun run(p, begin);
    // sixteen waves leave a lane 128 registers: no room for a row ahead at 16 features
    if constexpr (VEC && !(TW == 16 && EPL == 16)) {
        // The next token's arrays are on their way while one is worked on; the
        // vectors stay in registers as they are in memory.
        using Raw = RawRow<T, EPL, TW>;
        Raw w, pw, pb, gate, dy, r, dr, u;
        f32x4 st = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.dy != nullptr) w.load(p.weight, 0, p.d, l);
        if (POST) {
            pw.load(p.post_weight, 0, p.d, l);
            if (p.post_bias != nullptr) pb.load(p.post_bias, 0, p.d, l);
        }
        auto fetch = [&](int64_t n) {
            const int64_t off = n * p.d;
            if (p.dy != nullptr) {
                dy.load(p.dy, off, p.d, l);
                r.load(p.r, off, p.d, l);
            }
            if (p.dr != nullptr) dr.load(p.dr, off, p.d, l);
            if (p.need_u) u.load(p.branch, off, p.d, l);
            st = *reinterpret_cast<const f32x4*>(p.stats + 4 * n);
        };
        if (begin < end) {
            fetch(begin);
            if (GATE) gate.load(p.gate, run.row * p.d, p.d, l);
        }
        for (int64_t n = begin; n < end; ++n) {
            float vdy[EPL], vr[EPL], g[EPL], vu[EPL];
            if (p.dy != nullptr) {
                dy.get(vdy);
                r.get(vr);
            }
            if (p.dr != nullptr) dr.get(g);
            else clear(g);
            if (p.need_u) u.get(vu);
            const f32x4 s = st;
            if (n + 1 < end) fetch(n + 1);
            auto vec = [&](int k, float (&v)[EPL]) {
                if (k == 0) w.get(v);
                else if (k == 1) pw.get(v);
                else if (k == 2) pb.get(v);
                else gate.get(v);
            };
            auto store_dx = [&](const float (&v)[EPL]) {
                if (p.dx != nullptr) row_store<T, EPL, TW, VEC>(p.dx, n * p.d, p.d, l, v);
            };
            backward_row<EPL, POST, GATE>(p, s, vdy, vr, g, vu, acc, vec, sum, store_dx);
            if (p.dbranch != nullptr) row_store<T, EPL, TW, VEC>(p.dbranch, n * p.d, p.d, l, vu);
            if (GATE) {
                if (p.dgate != nullptr && (n + 1 == run.hi || n + 1 == end))
                    flush<T, EPL, TW, VEC>(p, team, begin, end, run, l, acc.v[kGateSum]);
                if (n + 1 == run.hi && n + 1 < end) {
                    run.next(p, n + 1);
                    gate.load(p.gate, run.row * p.d, p.d, l);
                }
            }
        }
    } else {
        for (int64_t n = begin; n < end; ++n) {
            float dy[EPL], r[EPL], g[EPL], u[EPL];
            const int64_t off = n * p.d;
            if (p.dy != nullptr) {
                row_load<T, EPL, TW, VEC>(p.dy, off, p.d, l, dy);
                row_load<T, EPL, TW, VEC>(p.r, off, p.d, l, r);
            }
            if (p.dr != nullptr) row_load<T, EPL, TW, VEC>(p.dr, off, p.d, l, g);
            else clear(g);
            if (p.need_u) row_load<T, EPL, TW, VEC>(p.branch, off, p.d, l, u);
            backward_token<T, EPL, TW, VEC, POST, GATE>(p, n, run.row, l, dy, r, g, u, acc, sum);
            if (p.dbranch != nullptr) row_store<T, EPL, TW, VEC>(p.dbranch, off, p.d, l, u);
            if (GATE) {
                if (p.dgate != nullptr && (n + 1 == run.hi || n + 1 == end))
                    flush<T, EPL, TW, VEC>(p, team, begin, end, run, l, acc.v[kGateSum]);
                run.next(p, n + 1);
            }
        }
    }
    if (p.arrays == 0) return;
    if (TW > 1) __syncthreads();
    write_partials<EPL, TW, VEC, kTeams>(p, blockIdx.x, mine, l, acc, sh);
}

// Feature-major dy or branch (and dbranch): TT tokens a workgroup, TT /
// kTileWaves consecutive ones a wave. dy's tile takes dbranch where the branch
// has none of its own.
template <class T, int EPL, int TT, bool VEC, bool POST, bool GATE>
__global__ __launch_bounds__(kTileThreads) void norm_backward_tile_kernel(const BwdRow p,
                                                                          int branch_cols,
                                                                          int y_cols, int pairs) {
    extern __shared__ float sh[];
    TeamSum<1, 2> sum{nullptr};
    const int l = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t group = xcd_logical_block(blockIdx.x, gridDim.x);
    const int64_t n0 = group * TT;
    const bool dy_tile = y_cols && p.dy != nullptr;
    const bool u_tile = branch_cols && p.need_u;
    float* ty = sh;
    float* tu = dy_tile && u_tile ? sh + 4 * tile_quarter(p.d) * (TT + 1) : sh;
    constexpr int kPer = TT / kTileWaves;
    const int64_t begin = n0 + wv * kPer;
    const int64_t end = begin + kPer < p.n ? begin + kPer : p.n;
    Ahead<T, EPL, VEC, (EPL == 16 && !POST)> ar, adr;
    auto fetch = [&](int64_t n) {
        if (p.dy != nullptr) ar.fetch(p.r, n * p.d, p.d, l);
        if (p.dr != nullptr) adr.fetch(p.dr, n * p.d, p.d, l);
    };
    if (begin < end) fetch(begin);
    if (dy_tile) tile_load<T, TT>(p.dy, p.n, p.d, n0, pairs, ty);
    if (u_tile) tile_load<T, TT>(p.branch, p.n, p.d, n0, pairs, tu);
    __syncthreads();
    const int64_t team = group * kTileWaves + wv;
    Acc<EPL> acc;
#pragma unroll
    for (int k = 0; k < kColSums; ++k) clear(acc.v[k]);
    GateRun run(p, begin);
#pragma unroll 1  // unrolled, the tokens' registers add up
    for (int64_t n = begin; n < end; ++n) {
        const int t = static_cast<int>(n - n0);
        float dy[EPL], r[EPL], g[EPL], u[EPL];
        const int64_t off = n * p.d;
        if (p.dy != nullptr) {
            ar.get(p.r, off, p.d, l, r);
            if (dy_tile) tile_row_load<EPL, TT, VEC>(ty, t, p.d, l, dy);
            else row_load<T, EPL, 1, VEC>(p.dy, off, p.d, l, dy);
        }
        if (p.dr != nullptr) adr.get(p.dr, off, p.d, l, g);
        else clear(g);
        if (n + 1 < end) fetch(n + 1);
        if (u_tile) tile_row_load<EPL, TT, VEC>(tu, t, p.d, l, u);
        else if (p.need_u) row_load<T, EPL, 1, VEC>(p.branch, off, p.d, l, u);
        backward_token<T, EPL, 1, VEC, POST, GATE>(p, n, run.row, l, dy, r, g, u, acc, sum);
        if (p.dbranch != nullptr) {
            if (branch_cols) tile_row_store<EPL, TT, VEC>(tu, t, p.d, l, u);
            else row_store<T, EPL, 1, VEC>(p.dbranch, off, p.d, l, u);
        }
        if (GATE) {
            if (p.dgate != nullptr && (n + 1 == run.hi || n + 1 == end))
                flush<T, EPL, 1, VEC>(p, team, begin, end, run, l, acc.v[kGateSum]);
            run.next(p, n + 1);
        }
    }
    __syncthreads();
    if (p.dbranch != nullptr && branch_cols) {
        tile_store<T, TT>(p.dbranch, p.n, p.d, n0, pairs, tu);
        __syncthreads();
    }
    if (p.arrays == 0) return;
    write_partials<EPL, 1, VEC, kTileWaves>(p, group, wv, l, acc, sh);
}

// out[c] = Σ over the partials of column c, in order: 64 columns a workgroup,
// 16 threads a column, each a run of consecutive partials.
struct ColSums {
    const float* partial;
    void* out[kColSums];  // the arrays that are there, in the partial's order
    int64_t groups;
    int arrays, d;
};

template <class T>
__global__ __launch_bounds__(1024) void norm_colsum_kernel(const ColSums p) {
    __shared__ float sh[16][kWave + 1];
    const int c = blockIdx.x * kWave + (threadIdx.x & (kWave - 1));
    const int part = threadIdx.x >> 6;
    const int width = p.arrays * p.d;
    const int64_t per = (p.groups + 15) / 16;
    const int64_t g0 = part * per, g1 = g0 + per < p.groups ? g0 + per : p.groups;
    float s = 0.0f;
    if (c < width) {
        int64_t g = g0;
        for (; g + 8 <= g1; g += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = p.partial[(g + j) * width + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; g < g1; ++g) s += p.partial[g * width + c];
    }
    sh[part][threadIdx.x & (kWave - 1)] = s;
    __syncthreads();
    if (part == 0 && c < width) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += sh[k][threadIdx.x];
        T::store(p.out[c / p.d], c % p.d, s);
    }
}

// dgate of a gate row whose tokens more than one team held: its teams' partial
// rows, in order; PARTS threads a column, each a run of consecutive teams.
template <class T, int PARTS>
__global__ __launch_bounds__(PARTS * kWave) void norm_gate_kernel(const BwdRow p) {
    __shared__ float sh[PARTS][kWave];
    const int64_t grp = blockIdx.x;
    const int64_t lo = grp * p.per_gate, hi = lo + p.per_gate;
    const int64_t t0 = lo / p.per_team, t1 = (hi - 1) / p.per_team;
    if (t0 == t1) return;  // written by its team
    const int c = threadIdx.x & (kWave - 1), part = threadIdx.x >> 6;
    const int e = blockIdx.y * kWave + c;
    const int64_t per = (t1 - t0 + PARTS) / PARTS;
    const int64_t a = t0 + part * per, b = a + per < t1 + 1 ? a + per : t1 + 1;
    float s = 0.0f;
    if (e < p.d) {
        // slot 0 of a team that began inside the run, slot 1 of the one it began in
        auto at = [&](int64_t t) {
            return p.gate_partial[(2 * t + (lo < t * p.per_team ? 0 : 1)) * p.d + e];
        };
        int64_t t = a;
        for (; t + 8 <= b; t += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = at(t + j);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; t < b; ++t) s += at(t);
    }
    if (PARTS > 1) {
        sh[part][c] = s;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int k = 1; k < PARTS; ++k) s += sh[k][c];
    }
    if (e < p.d) T::store(p.dgate, grp * p.d + e, s);
}

// Teams and workgroups of a backward, and its workspace.
struct Plan {
    int tw;            // waves of a team
    int tile;          // tokens of a workgroup's tile, 0: the row kernels
    int64_t per_team;  // tokens of a team
    int64_t groups;    // workgroups
    int64_t teams;
    int arrays;
    int at[kColSums];
    bool gate_all, gate_some;  // dgate as a sum over all tokens / over some
    int64_t bytes() const {
        return 4 * (groups * arrays * d + (gate_some ? 2 * teams * d : 0));
    }
    int64_t d;
};

// Workgroups that share the tokens: enough to fill the card twice over, few
// enough that their partial rows cost little beside the arrays themselves.
constexpr int64_t kBwdGroups = 512;

// Whether the branch itself is read (else only its gradient is written).
bool needs_branch(const slk_norm* a) {
    return a->branch != nullptr && (a->post_weight != nullptr ||
                                    (a->gate != nullptr && a->dgate != nullptr));
}

Plan make_plan(const slk_norm* a) {
    Plan p;
    p.d = a->d;
    const bool want_gate = a->dgate != nullptr && a->gate != nullptr;
    p.gate_all = want_gate && a->gate_rows == 1;
    p.gate_some = want_gate && a->gate_rows > 1 && a->gate_rows < a->n;
    const bool wanted[kColSums] = {a->dweight != nullptr && a->dy != nullptr,
                                   a->dbias != nullptr && a->dy != nullptr,
                                   a->dpost_weight != nullptr, a->dpost_bias != nullptr,
                                   p.gate_all};
    p.arrays = 0;
    for (int k = 0; k < kColSums; ++k) p.at[k] = wanted[k] ? p.arrays++ : -1;
    const bool cols = (a->branch_cols && a->branch != nullptr) || a->y_cols;
    const bool both = a->branch_cols && needs_branch(a) && a->y_cols && a->dy != nullptr;
    p.tile = cols ? tile_tokens(a->n, a->d, (both ? 75 : 150) * 1024) : 0;
    if (p.tile) {
        p.tw = 1;
        p.per_team = p.tile / kTileWaves;
        p.groups = ceil_div(a->n, p.tile);
        p.teams = p.groups * kTileWaves;
        return p;
    }
    norm_shape(static_cast<int>(a->d), [&](auto, auto tw) { p.tw = decltype(tw)::value; });
    const int64_t teams_per_group = p.tw == 1 ? kNormThreads / kWave : 1;
    const int64_t want = p.tw >= 8 ? kBwdGroups / 2 : kBwdGroups;
    p.per_team = ceil_div(a->n, want * teams_per_group);
    if (p.per_team < 1) p.per_team = 1;
    p.groups = ceil_div(a->n, p.per_team * teams_per_group);
    p.teams = p.groups * teams_per_group;
    return p;
}

template <class T, bool POST, bool GATE>
int backward(const slk_norm* a, const Plan& plan, const BwdRow& p, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(plan.groups));
    if (plan.tile) {
        const bool dy_tile = a->y_cols && p.dy != nullptr, u_tile = a->branch_cols && p.need_u;
        const size_t tiles = dy_tile && u_tile ? 2 : 1;
        const size_t lds = tiles * 4 * tile_quarter(p.d) * (plan.tile + 1) * sizeof(float);
        const int pairs = tile_pairs(a, {dy_tile ? a->dy : nullptr, u_tile ? a->branch : nullptr,
                                         a->branch_cols ? a->dbranch : nullptr});
        const bool vec = norm_vec(a, {a->r, a->branch_cols ? nullptr : a->branch, a->gate,
                                      a->weight, a->post_weight, a->post_bias, a->dr,
                                      a->y_cols ? nullptr : a->dy, a->dx,
                                      a->branch_cols ? nullptr : a->dbranch, a->dgate});
        auto go = [&](auto kv, auto ks) {
            if (vec) {
                hipLaunchKernelGGL(kv, grid, dim3(kTileThreads), lds, st, p, a->branch_cols,
                                   a->y_cols, pairs);
            } else {
                hipLaunchKernelGGL(ks, grid, dim3(kTileThreads), lds, st, p, a->branch_cols,
                                   a->y_cols, pairs);
            }
        };
        auto pick = [&](auto epl, auto tt) {
            constexpr int E = decltype(epl)::value, TT = decltype(tt)::value;
            go(norm_backward_tile_kernel<T, E, TT, true, POST, GATE>,
               norm_backward_tile_kernel<T, E, TT, false, POST, GATE>);
        };
        using std::integral_constant;
        if (p.d <= 512 && plan.tile == 32) pick(integral_constant<int, 8>{}, integral_constant<int, 32>{});
        else if (p.d <= 512) pick(integral_constant<int, 8>{}, integral_constant<int, 16>{});
        else if (plan.tile == 32) pick(integral_constant<int, 16>{}, integral_constant<int, 32>{});
        else pick(integral_constant<int, 16>{}, integral_constant<int, 16>{});
        return check_launch("norm_backward");
    }
    const bool vec = norm_vec(a, {a->r, a->branch, a->gate, a->weight, a->post_weight,
                                  a->post_bias, a->dr, a->dy, a->dx, a->dbranch, a->dgate});
    auto go = [&](auto kv, auto ks, int threads, size_t lds) {
        if (vec) hipLaunchKernelGGL(kv, grid, dim3(threads), lds, st, p);
        else hipLaunchKernelGGL(ks, grid, dim3(threads), lds, st, p);
    };
    auto pick = [&](auto epl, auto tw) {
        constexpr int E = decltype(epl)::value, W = decltype(tw)::value;
        const size_t lds = W == 1 ? static_cast<size_t>(kNormThreads / kWave) * p.d * sizeof(float)
                                  : 4 * W * sizeof(float);
        go(norm_backward_kernel<T, E, W, true, POST, GATE>,
           norm_backward_kernel<T, E, W, false, POST, GATE>, W == 1 ? kNormThreads : W * kWave,
           lds);
    };
    norm_shape(p.d, pick);
    return check_launch("norm_backward");
}

template <class T>
int backward_any(const slk_norm* a, const Plan& plan, const BwdRow& p, hipStream_t st) {
    const bool post = a->post_weight != nullptr, gate = a->gate != nullptr;
    int rc = post ? (gate ? backward<T, true, true>(a, plan, p, st)
                          : backward<T, true, false>(a, plan, p, st))
                  : (gate ? backward<T, false, true>(a, plan, p, st)
                          : backward<T, false, false>(a, plan, p, st));
    if (rc != SLK_OK) return rc;
    if (plan.arrays > 0) {
        ColSums c;
        void* outs[kColSums] = {a->dweight, a->dbias, a->dpost_weight, a->dpost_bias, a->dgate};
        for (int k = 0; k < kColSums; ++k)
            if (plan.at[k] >= 0) c.out[plan.at[k]] = outs[k];
        c.partial = p.partial;
        c.groups = plan.groups;
        c.arrays = plan.arrays;
        c.d = p.d;
        hipLaunchKernelGGL(norm_colsum_kernel<T>,
                           dim3(static_cast<unsigned>(ceil_div(plan.arrays * p.d, kWave))),
                           dim3(1024), 0, st, c);
        rc = check_launch("norm_backward sums");
        if (rc != SLK_OK) return rc;
    }
    if (plan.gate_some) {
        const dim3 grid(static_cast<unsigned>(a->gate_rows),
                        static_cast<unsigned>(ceil_div(p.d, kWave)));
        if (p.per_gate >= 32 * p.per_team) {
            hipLaunchKernelGGL((norm_gate_kernel<T, 16>), grid, dim3(16 * kWave), 0, st, p);
        } else {
            hipLaunchKernelGGL((norm_gate_kernel<T, 1>), grid, dim3(kWave), 0, st, p);
        }
        rc = check_launch("norm_backward gate");
    }
    return rc;
}

}  // namespace
}  // namespace slk

extern "C" int64_t slk_norm_workspace_bytes(const slk_norm* a) {
    using namespace slk;
    clear_error();
    if (a == nullptr || a->n <= 0 || a->d < 1 || a->d > SLK_NORM_MAX_D) return 0;
    return make_plan(a).bytes();
}

extern "C" int slk_norm_backward(const slk_norm* a, void* stream) {
    using namespace slk;
    clear_error();
    const int rc = validate_norm(a, "norm_backward", true);
    if (rc != SLK_OK) return rc;
    if (a->n == 0) return SLK_OK;
    if ((a->dgate != nullptr || a->dpost_weight != nullptr || a->dpost_bias != nullptr ||
         a->dbranch != nullptr) && a->branch == nullptr) {
        return fail(SLK_EINVAL, "norm_backward: a branch's gradient without a branch");
    }
    const Plan plan = make_plan(a);
    if (plan.bytes() > a->workspace_bytes || (plan.bytes() > 0 && a->workspace == nullptr)) {
        return fail(SLK_EINVAL, "norm_backward: workspace too small: " +
                                    std::to_string(a->workspace_bytes) + " < " +
                                    std::to_string(plan.bytes()));
    }
    BwdRow p;
    p.r = a->r;
    p.gate = a->gate;
    p.weight = a->weight;
    p.post_weight = a->post_weight;
    p.post_bias = a->post_bias;
    p.dr = a->dr;
    p.dy = a->dy;
    p.branch = a->branch;
    p.dx = a->dx;
    p.dbranch = a->dbranch;
    p.dgate = plan.gate_all ? nullptr : a->dgate;
    p.stats = a->stats;
    p.partial = static_cast<float*>(a->workspace);
    p.gate_partial = p.partial + plan.groups * plan.arrays * a->d;
    p.n = a->n;
    p.per_gate = a->gate != nullptr ? a->n / a->gate_rows : 1;
    p.per_team = plan.per_team;
    p.d = static_cast<int>(a->d);
    p.arrays = plan.arrays;
    for (int k = 0; k < kColSums; ++k) p.at[k] = plan.at[k];
    p.layer = a->layer != 0;
    p.need_u = needs_branch(a);
    p.scale = static_cast<float>(a->scale);
    p.inv_d = 1.0f / static_cast<float>(a->d);
    return a->dtype == SLK_F32 ? backward_any<F32>(a, plan, p, as_stream(stream))
                               : backward_any<BF16>(a, plan, p, as_stream(stream));
}
