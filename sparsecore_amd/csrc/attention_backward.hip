// slk_attention_backward's kernels: one computes dK and dV for a block of keys
// over the queries that see it, the other dQ (and the bias's gradient) for a
// block of queries over the keys that they see. Each recomputes the weights from
// the forward's log-sums: seven products where five would do with sums of dQ
// through atomics, whose order would change the results from run to run.
#include "attention.hpp"
#include "elem.hpp"

namespace slk {

namespace {

// Exponent above the largest |dS| of a pair of tiles: |dP| < DP·2^(oe + 1)·2^(ve + 1), and
// |delta| < 2^(de + 1).
__device__ __forceinline__ int ds_exponent(int oe, int ve, int de, int log_dp) {
    return min(max(max(oe + ve + log_dp + 2, de + 1) + 1, -100), 100);
}

__device__ __forceinline__ int wave_max(int e) {
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) e = max(e, __shfl_xor(e, x));
    return __builtin_amdgcn_readfirstlane(e);
}

// 64 floats of a row array into LDS, by one wave.
__device__ __forceinline__ void load_row(const float* from, unsigned char* to, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint64_t at = reinterpret_cast<uint64_t>(from);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    const char* src = reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
    uint32_t o = 4 * lane;
    asm("" : "+v"(o));
    __builtin_amdgcn_global_load_lds(src + o, to, 4, 0, 0);
#else
    (void)from, (void)to, (void)lane;
#endif
}

// dK, dV: a workgroup takes 128 keys of one key head, a wave 32 of them, whose
// rows of K and V stay in registers. Q and dO come through LDS, 64 rows at a
// time, for every query head of the group in turn. Scores are Q·K^T here: a lane
// holds 16 queries of one key, as the operands of dV^T = dO^T·P and
// dK^T = Q^T·dS need them.
template <bool SPLIT, int DB, bool BIAS>
__global__ __launch_bounds__(kAttnThreads, DB * (SPLIT ? 2 : 1) <= 4 ? 2 : 1) void
attn_dkv_kernel(const AttnArgs g) {
    using T = AttnTile<DB>;
    constexpr int kBytes = (SPLIT ? 2 : 1) * T::kPlane, KS = 2 * DB;
    constexpr int kLogDp = DB == 1 ? 5 : DB == 2 ? 6 : 7;
    __shared__ __align__(16) unsigned char ring0[2 * kBytes + 512];
    __shared__ __align__(16) unsigned char ring1[2 * kBytes + 512];
    extern __shared__ float bias_row[];

    const int t = threadIdx.x, lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const int rep = g.heads / g.kv_heads;
    const int kvh = blockIdx.x % g.kv_heads;
    int sid, tile;
    if (!attn_entry(g.plan, blockIdx.x / g.kv_heads, g.tiles, true, sid, tile)) return;
    const AttnSeq seq = attn_seq(g.plan, sid);
    const int shift = seq.nk - seq.nq;
    const int key0 = tile * 128 + 32 * wv, key = key0 + (lane & 31);

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int fb = 0; fb < DB; ++fb)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[fb][r] = dv[fb][r] = 0.0f;
    int co = 0, cq = 0;

    // tiles of 64 queries, from the first that sees a key of the workgroup
    const int first = g.causal ? max(0, tile * 128 - shift) / kAttnRows : 0;
    const int n_q = (seq.nq + kAttnRows - 1) / kAttnRows;
    const int nt = tile * 128 < seq.nk && first < n_q ? n_q - first : 0;

    if (nt > 0) {
        const int64_t q0_tile = seq.pq / 64 + first;
        auto issue = [&](unsigned char* to, int hr, int qt) __attribute__((always_inline)) {
            const int head = kvh * rep + hr;
            const int64_t at = (q0_tile + qt) * kBytes;
            attn_stage<kBytes>(g.q.p + head * g.q.sh + at, to, wv, lane);
            attn_stage<kBytes>(g.dout.p + head * g.dout.sh + at, to + kBytes, wv, lane);
            const int64_t row = head * g.lse_sh + (q0_tile + qt) * 64;
            if (wv == 0) load_row(g.lse + row, to + 2 * kBytes, lane);
            if (wv == 1) load_row(g.delta + row, to + 2 * kBytes + 256, lane);
        };
        issue(ring0, 0, 0);
        const AttnReads<SPLIT, DB> rd(lane);

        const bool live = key0 < seq.nk;
        const int k_row = seq.pk + (live ? key0 : 0);
        AttnPair<SPLIT> kf[KS], vf[KS];
        {
            const int64_t at = static_cast<int64_t>(k_row / 64) * kBytes;
            const unsigned char* ka =
                reinterpret_cast<const unsigned char*>(g.k.p + kvh * g.k.sh + at);
            const unsigned char* va =
                reinterpret_cast<const unsigned char*>(g.v.p + kvh * g.v.sh + at);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kf[ks] = rd.along(ka, (k_row >> 5) & 1, ks);
                vf[ks] = rd.along(va, (k_row >> 5) & 1, ks);
            }
        }
        // dV in units of 2^(co - 28), dK of 2^(cq - 28), the largest of the query
        // tiles that this wave's keys are seen by
        const int ke = attn_exp(g.k, kvh, k_row), ve = attn_exp(g.v, kvh, k_row);
        co = cq = -400;
        {
            const int b0 = g.causal ? max(0, key0 - shift) / 64 : 0;
            for (int hr = 0; hr < rep; ++hr) {
                const int64_t at = (kvh * rep + hr) * g.q.exps_sh + seq.pq / 64;
                for (int i = b0 + lane; i < n_q; i += 64) {
                    const int oe = g.dout.exps[at + i] >> 1;
                    co = max(co, oe);
                    cq = max(cq, ds_exponent(oe, ve, g.dexps[at + i], kLogDp) +
                                     (g.q.exps[at + i] >> 1));
                }
            }
            co = wave_max(co);
            cq = wave_max(cq);
        }
        const int md = BIAS ? g.bias.max_distance : 0;

        auto compute = [&](const unsigned char* buf, int hr, int q_tile)
            __attribute__((always_inline)) {
            const int head = kvh * rep + hr, row0 = seq.pq + q_tile;
            const int qe = attn_exp(g.q, head, row0), oe = attn_exp(g.dout, head, row0);
            const int de = __builtin_amdgcn_readfirstlane(
                g.dexps[head * g.q.exps_sh + (row0 >> 6)]);
            const float c = ldexpf(g.scale2, qe + ke - 2 * kAttnUnit);
            // weights times 2^u; dS = weight · (alpha·dp - beta·delta)
            const int u = kAttnUnit + max(oe - co, -60);
            const int b = ds_exponent(oe, ve, de, kLogDp);
            const int x = kAttnUnit - b + max(b + qe - cq, -60) - u;
            const float unit = static_cast<float>(u);
            const float alpha = attn_pow2(x + oe + ve - 2 * kAttnUnit), beta = attn_pow2(x);
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                const int q0 = q_tile + 32 * qb;
                if (q0 >= seq.nq || (g.causal && q0 + 31 + shift < key0)) continue;
                const bool masked = q0 + 31 >= seq.nq || (g.causal && q0 + shift < key0 + 31);
                f32x16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    s = attn_dot<SPLIT>(rd.along(buf, qb, ks), kf[ks], s);
                    dp = attn_dot<SPLIT>(rd.along(buf + kBytes, qb, ks), vf[ks], dp);
                }
                const float* lse = reinterpret_cast<const float*>(buf + 2 * kBytes) + 32 * qb;
                const float* delta = lse + 64;
                float p[16], ds[16];
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int row = 8 * r4 + 4 * (lane >> 5);
                    const f32x4 z = *reinterpret_cast<const f32x4*>(lse + row);
                    const f32x4 d = *reinterpret_cast<const f32x4*>(delta + row);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 4 * r4 + j;
                        float add = unit - z[j];
                        if constexpr (BIAS)
                            add += bias_row[md + attn_clamp(q0 + row + j + shift - key, md)];
                        p[r] = attn_exp2(__builtin_fmaf(s[r], c, add));
                        ds[r] = p[r] * __builtin_fmaf(dp[r], alpha, -(d[j] * beta));
                    }
                }
                // the lane's key is seen by rows [lo, hi) of the block
                const int lo = g.causal ? key - shift - q0 : 0, hi = seq.nq - q0;
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int row = attn_row(r, lane);
                        const bool see = row >= lo && row < hi;
                        p[r] = see ? p[r] : 0.0f;
                        ds[r] = see ? ds[r] : 0.0f;
                    }
                }
                AttnPair<SPLIT> wp[2] = {attn_operand<SPLIT>(p), attn_operand<SPLIT>(p + 8)};
                AttnPair<SPLIT> wd[2] = {attn_operand<SPLIT>(ds), attn_operand<SPLIT>(ds + 8)};
                attn_accumulate<SPLIT, DB>(rd, buf + kBytes, qb, wp, dv);
                attn_accumulate<SPLIT, DB>(rd, buf, qb, wd, dk);
            }
        };
        int hr = 0, qt = 0;
        auto stage = [&](const unsigned char* cur, unsigned char* next)
            __attribute__((always_inline)) {
            const int h = hr, i = qt;
            if (++qt == nt) {
                qt = 0;
                ++hr;
            }
            __builtin_amdgcn_s_waitcnt(wait_vm(0));
            asm volatile("s_barrier" ::: "memory");
            if (hr < rep) issue(next, hr, qt);
            if (BIAS && i == 0) {  // a head's first tile
                attn_bias_row(g.bias, kvh * rep + h, bias_row);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            if (live) compute(cur, h, (first + i) * kAttnRows);
        };
        int left = rep * nt;
        for (; left >= 2; left -= 2) {
            stage(ring0, ring1);
            stage(ring1, ring0);
        }
        if (left) stage(ring0, ring1);
    }

    if (key >= seq.ek) return;
    const float fk = ldexpf(g.scale, cq - 2 * kAttnUnit), fv = attn_pow2(co - 2 * kAttnUnit);
    const bool zero = key >= seq.nk || nt == 0;
    const AttnIo* const to[2] = {&g.dk, &g.dv};
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const AttnIo& io = *to[which];
        const int64_t at = sid * io.sb + (seq.k0 + key) * io.sr + kvh * io.sh;
        const bool vec = io.sd == 1 && g.vec_kv;
#pragma unroll
        for (int fb = 0; fb < DB; ++fb) {
            f32x16 x = which ? dv[fb] : dk[fb];
            if (zero) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 0.0f;
            }
            const float f = zero ? 1.0f : which ? fv : fk;
            if (g.dtype == SLK_F32) attn_store<F32>(io, at, fb, lane, g.dim, vec, x, f);
            else attn_store<BF16>(io, at, fb, lane, g.dim, vec, x, f);
        }
    }
}

// dQ: a workgroup takes 128 queries of one head, a wave 32 of them, whose rows of
// Q and dO stay in registers; K and V come through LDS. The bias's gradient: each
// wave half adds a lane's dS to bins of its own, one a distance (for one register
// the 32 lanes' distances differ), so the sums need no atomicity and repeat.
template <bool SPLIT, int DB, bool BIAS>
__global__ __launch_bounds__(kAttnThreads, DB * (SPLIT ? 2 : 1) <= 4 ? 2 : 1) void
attn_dq_kernel(const AttnArgs g) {
    using T = AttnTile<DB>;
    constexpr int kBytes = (SPLIT ? 2 : 1) * T::kPlane, KS = 2 * DB;
    constexpr int kLogDp = DB == 1 ? 5 : DB == 2 ? 6 : 7;
    __shared__ __align__(16) unsigned char ring0[2 * kBytes];
    __shared__ __align__(16) unsigned char ring1[2 * kBytes];
    extern __shared__ float bias_row[];

    const int t = threadIdx.x, lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t rep = g.heads / g.kv_heads;
    const uint32_t kvh = blockIdx.x % g.kv_heads, u0 = blockIdx.x / g.kv_heads;
    const int head = static_cast<int>(kvh * rep + u0 % rep);
    int sid, tile;
    if (!attn_entry(g.plan, u0 / rep, g.tiles, false, sid, tile)) return;
    const AttnSeq seq = attn_seq(g.plan, sid);
    const int rows0 = tile * 128, shift = seq.nk - seq.nq;
    const int wave0 = rows0 + 32 * wv;
    const int q = wave0 + (lane & 31);
    const int last_q = min(rows0 + 128, seq.nq) - 1;
    const int seen = last_q < rows0 ? 0 : g.causal ? min(seq.nk, last_q + shift + 1) : seq.nk;
    const int t1 = seen <= 0 ? 0 : (seen + kAttnRows - 1) / kAttnRows;

    const int md = BIAS ? g.bias.max_distance : 0, width = 2 * md + 1;
    float* const bins = bias_row + width;        // [wave][half][distance]
    float* const far = bins + 8 * width;         // [wave][below, above]
    float below = 0.0f, above = 0.0f;            // distances past the last bins
    if constexpr (BIAS) {
        attn_bias_row(g.bias, head, bias_row);
        for (int i = t; i < 8 * width; i += kAttnThreads) bins[i] = 0.0f;
    }

    f32x16 dq[DB];
#pragma unroll
    for (int fb = 0; fb < DB; ++fb)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[fb][r] = 0.0f;
    int ck = 0;

    if (t1 > 0) {
        const int64_t k_tile = seq.pk / 64;
        auto issue = [&](unsigned char* to, int kt) __attribute__((always_inline)) {
            const int64_t at = (k_tile + kt) * kBytes;
            attn_stage<kBytes>(g.k.p + kvh * g.k.sh + at, to, wv, lane);
            attn_stage<kBytes>(g.v.p + kvh * g.v.sh + at, to + kBytes, wv, lane);
        };
        issue(ring0, 0);
        const AttnReads<SPLIT, DB> rd(lane);

        const int q_row = seq.pq + min(wave0, (seq.nq + 63) / 64 * 64 - 32);
        AttnPair<SPLIT> qf[KS], of[KS];
        {
            const int64_t at = static_cast<int64_t>(q_row / 64) * kBytes;
            const unsigned char* qa =
                reinterpret_cast<const unsigned char*>(g.q.p + head * g.q.sh + at);
            const unsigned char* oa =
                reinterpret_cast<const unsigned char*>(g.dout.p + head * g.dout.sh + at);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qf[ks] = rd.along(qa, (q_row >> 5) & 1, ks);
                of[ks] = rd.along(oa, (q_row >> 5) & 1, ks);
            }
        }
        const bool mine = q < seq.nq;
        const int64_t ri = head * g.lse_sh + q_row + (lane & 31);
        const float lse = mine ? g.lse[ri] : INFINITY;
        const float delta = mine ? g.delta[ri] : 0.0f;
        const int qe = attn_exp(g.q, head, q_row), oe = attn_exp(g.dout, head, q_row);
        const int de =
            __builtin_amdgcn_readfirstlane(g.dexps[head * g.q.exps_sh + (q_row >> 6)]);
        {
            const int* ve = g.v.exps + kvh * g.v.exps_sh + k_tile;
            const int* ke = g.k.exps + kvh * g.k.exps_sh + k_tile;
            int e = -400;
            for (int i = lane; i < t1; i += 64)
                e = max(e, ds_exponent(oe, ve[i] >> 1, de, kLogDp) + (ke[i] >> 1));
            ck = wave_max(e);
        }

        auto compute = [&](const unsigned char* buf, int key_tile) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key0 = key_tile + 32 * kb;
                if (key0 >= seq.nk) return;
                if (g.causal && key0 > wave0 + 31 + shift) return;
                const bool masked =
                    key0 + 31 >= seq.nk || (g.causal && key0 + 31 > wave0 + shift);
                const int ke = attn_exp(g.k, kvh, seq.pk + key0);
                const int ve = attn_exp(g.v, kvh, seq.pk + key0);
                const float c = ldexpf(g.scale2, qe + ke - 2 * kAttnUnit);
                const int b = ds_exponent(oe, ve, de, kLogDp);
                const int x = kAttnUnit - b + max(b + ke - ck, -60);
                const float alpha = attn_pow2(x + oe + ve - 2 * kAttnUnit);
                const float db = delta * attn_pow2(x);
                f32x16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    s = attn_dot<SPLIT>(rd.along(buf, kb, ks), qf[ks], s);
                    dp = attn_dot<SPLIT>(rd.along(buf + kBytes, kb, ks), of[ks], dp);
                }
                const int lim = (g.causal ? min(seq.nk - 1, q + shift) : seq.nk - 1) - key0;
                const int away = q + shift - key0;
                bool near = false;
                float flat = 0.0f;
                if constexpr (BIAS) {
                    const int lo = wave0 + shift - key0 - 31, hi = lo + 62;
                    near = lo < md && hi > -md;
                    flat = bias_row[lo >= md ? 2 * md : 0];
                }
                float ds[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float add = -lse;
                    if constexpr (BIAS)
                        add += near ? bias_row[md + attn_clamp(away - attn_row(r, lane), md)]
                                    : flat;
                    const float p = attn_exp2(__builtin_fmaf(s[r], c, add));
                    ds[r] = p * __builtin_fmaf(dp[r], alpha, -db);
                }
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        ds[r] = attn_row(r, lane) <= lim ? ds[r] : 0.0f;
                }
                if constexpr (BIAS) {
                    const float back = attn_pow2(-x);
                    if (near) {
                        float* const mine_bins = bins + (2 * wv + (lane >> 5)) * width + md;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int d = away - attn_row(r, lane);
                            const float y = mine ? ds[r] * back : 0.0f;
                            if (d >= md) above += y;
                            else if (d <= -md) below += y;
                            else
                                __hip_atomic_fetch_add(mine_bins + d, y, __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_WORKGROUP);
                        }
                    } else {
                        float y = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) y += ds[r];
                        y = mine ? y * back : 0.0f;
                        if (away >= md) above += y;
                        else below += y;
                    }
                }
                AttnPair<SPLIT> w[2] = {attn_operand<SPLIT>(ds), attn_operand<SPLIT>(ds + 8)};
                attn_accumulate<SPLIT, DB>(rd, buf, kb, w, dq);
            }
        };
        auto stage = [&](const unsigned char* cur, unsigned char* next, int kt) __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(wait_vm(0));
            asm volatile("s_barrier" ::: "memory");
            if (kt + 1 < t1) issue(next, kt + 1);
            if (wave0 < seq.nq) compute(cur, kt * kAttnRows);
        };
        int kt = 0;
        for (; kt + 2 <= t1; kt += 2) {
            stage(ring0, ring1, kt);
            stage(ring1, ring0, kt + 1);
        }
        if (kt < t1) stage(ring0, ring1, kt);
    }

    if (q < seq.eq && g.dq.p != nullptr) {
        const bool zero = q >= seq.nq || t1 == 0;
        const float f = zero ? 1.0f : ldexpf(g.scale, ck - 2 * kAttnUnit);
        const int64_t at = sid * g.dq.sb + (seq.q0 + q) * g.dq.sr + head * g.dq.sh;
        const bool vec = g.dq.sd == 1 && g.vec_q;
#pragma unroll
        for (int fb = 0; fb < DB; ++fb) {
            f32x16 x = dq[fb];
            if (zero) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 0.0f;
            }
            if (g.dtype == SLK_F32) attn_store<F32>(g.dq, at, fb, lane, g.dim, vec, x, f);
            else attn_store<BF16>(g.dq, at, fb, lane, g.dim, vec, x, f);
        }
    }
    if constexpr (BIAS) {
        if (g.dbias_part == nullptr || rows0 >= seq.nq) return;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) {
            below += __shfl_xor(below, x);
            above += __shfl_xor(above, x);
        }
        if (lane == 0) {
            far[2 * wv] = below;
            far[2 * wv + 1] = above;
        }
        __syncthreads();
        const int slot = (seq.pq + rows0) / kAttnRows;
        const int slots = (seq.nq - rows0 + kAttnRows - 1) / kAttnRows;  // of this sequence, left
        float* const out = g.dbias_part + (head * g.dbias_slots + slot) * static_cast<int64_t>(width);
        for (int i = t; i < width; i += kAttnThreads) {
            float y = 0.0f;
            for (int j = 0; j < 8; ++j) y += bins[j * width + i];
            for (int j = 0; j < 4; ++j) y += i == 0 ? far[2 * j] : i == 2 * md ? far[2 * j + 1] : 0.0f;
            out[i] = y;
            if (slots > 1) out[width + i] = 0.0f;
        }
    }
}

// The bias's gradient from the workgroups' bins, in their order: a workgroup a
// head, a thread a distance, then a thread a bucket.
__global__ __launch_bounds__(1024) void attn_dbias_kernel(const AttnArgs g, void* dbias) {
    __shared__ float per[2 * SLK_ATTN_MAX_DISTANCE + 1];
    const int head = blockIdx.x, md = g.bias.max_distance, width = 2 * md + 1;
    const int64_t rows = g.plan.seqs != nullptr ? g.plan.count[1] : g.plan.batch * g.plan.pad_t;
    const int64_t slots = rows / kAttnRows;
    const float* from = g.dbias_part + head * g.dbias_slots * width;
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = 0.0f;
        int64_t s = 0;
        for (; s + 8 <= slots; s += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] += from[(s + j) * width + i];
        }
        for (; s < slots; ++s) y[0] += from[s * width + i];
        per[i] = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
    }
    __syncthreads();
    const int one = g.bias.one_sided ? g.bias.buckets : g.bias.buckets / 2;
    for (int b = threadIdx.x; b < g.bias.buckets; b += blockDim.x) {
        const int k = b < one ? b : b - one, step = b < one ? 1 : -1;
        const int n0 = g.bias.starts[k], n1 = k + 1 < one ? g.bias.starts[k + 1] : md + 1;
        float y = 0.0f;
        for (int n = n0; n < min(n1, md + 1); ++n)
            if (b < one || n > 0) y += per[md + step * n];
        const int64_t at = static_cast<int64_t>(b) * g.heads + head;
        if (g.bias.dtype == SLK_F32) F32::store(dbias, at, y);
        else BF16::store(dbias, at, y);
    }
}

template <bool SPLIT, int DB, bool BIAS>
int launch(const AttnArgs& g, const AttnPlan& kplan, int64_t q_entries, int64_t k_entries,
           bool want_q, bool want_kv, int64_t k_tiles, hipStream_t st) {
    const size_t width = BIAS ? 2 * g.bias.max_distance + 1 : 0;
    if (q_entries * g.heads > max_groups(kAttnThreads) ||
        k_entries * g.kv_heads > max_groups(kAttnThreads))
        return fail(SLK_EINVAL, "attention_backward: too many tiles");
    if (want_kv) {
        AttnArgs a = g;
        a.plan = kplan;
        a.tiles = k_tiles;
        hipLaunchKernelGGL((attn_dkv_kernel<SPLIT, DB, BIAS>),
                           dim3(static_cast<unsigned>(k_entries * g.kv_heads)),
                           dim3(kAttnThreads), width * sizeof(float), st, a);
        const int rc = check_launch("attention_backward: dk, dv");
        if (rc != SLK_OK) return rc;
    }
    if (want_q) {
        hipLaunchKernelGGL((attn_dq_kernel<SPLIT, DB, BIAS>),
                           dim3(static_cast<unsigned>(q_entries * g.heads)), dim3(kAttnThreads),
                           (9 * width + (BIAS ? 8 : 0)) * sizeof(float), st, g);
        return check_launch("attention_backward: dq");
    }
    return SLK_OK;
}

template <bool SPLIT, int DB>
int launch_bias(const AttnArgs& g, const AttnPlan& kplan, int64_t q_entries, int64_t k_entries,
                bool want_q, bool want_kv, int64_t k_tiles, hipStream_t st) {
    return g.bias.table != nullptr
               ? launch<SPLIT, DB, true>(g, kplan, q_entries, k_entries, want_q, want_kv, k_tiles,
                                         st)
               : launch<SPLIT, DB, false>(g, kplan, q_entries, k_entries, want_q, want_kv,
                                          k_tiles, st);
}

}  // namespace

int attn_launch_backward(const AttnArgs& g, bool split, int db, const AttnPlan& kplan,
                         int64_t q_entries, int64_t k_entries, bool want_q, bool want_kv,
                         int64_t k_tiles, hipStream_t st) {
    auto run = [&](auto f) { return f(g, kplan, q_entries, k_entries, want_q, want_kv, k_tiles, st); };
    if (split)
        return db == 1   ? run(launch_bias<true, 1>)
               : db == 2 ? run(launch_bias<true, 2>)
                         : run(launch_bias<true, 4>);
    return db == 1   ? run(launch_bias<false, 1>)
           : db == 2 ? run(launch_bias<false, 2>)
                     : run(launch_bias<false, 4>);
}

int attn_launch_dbias(const AttnArgs& g, void* dbias, hipStream_t st) {
    hipLaunchKernelGGL(attn_dbias_kernel, dim3(g.heads), dim3(1024), 0, st, g, dbias);
    return check_launch("attention_backward: bias");
}

}  // namespace slk
