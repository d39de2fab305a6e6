// slk_attention_backward's kernels: one computes dK and dV for a block of keys
// over the queries that see it, the other dQ (and the bias's gradient) for a
// block of queries over the keys that they see. Each recomputes the weights from
// the forward's log-sums: seven products where five would do with sums of dQ
// through atomics, whose order would change the results from run to run.
#include "attention.hpp"
#include "elem.hpp"

namespace slk {

namespace {

// dS as a float16 operand. Its parts reach 2^-24, so it is scaled to the size that it has,
// not to what it might have: a weight of 1 / keys and a dP far below its bound would leave
// 16 of 22 bits at 8192 keys. Each result row (a lane's) has a unit 2^c of its own; dS goes
// into the product times 2^(14 + e - c), e the exponent of the other operand's rows. Where
// a row's largest passes 2^kDsMost, or is below 2^kDsLeast so far, the unit is moved so
// that it comes to 2^kDsStart, and the sums with it, by powers of two (as the softmax's
// maximum is raised): in the first tile, and seldom after it. Before that a bound sees to
// it that nothing leaves float32: |dP - delta| < 2^b scaled stays below 2^kDsReach. That
// is looked at only where a tile's exponents differ from those it was looked at for.
constexpr int kDsMost = 15, kDsStart = 7, kDsLeast = 4, kDsReach = 80;

// Exponent above |dP| < DP·2^(oe + 1)·2^(ve + 1) and |delta| < 2^(de + 1), and their
// difference. Not below -20: powers of two from it stay in float32.
__device__ __forceinline__ int ds_exponent(int oe, int ve, int de, int log_dp) {
    return min(max(max(oe + ve + log_dp + 2, de + 1) + 1, -20), 120);
}

// Whether the largest scaled dS of some lane's row is out of range (0: none so far).
__device__ __forceinline__ bool ds_out(float most) {
    // no branches
    return (most > static_cast<float>(1 << kDsMost)) |
           ((most > 0.0f) & (most < static_cast<float>(1 << kDsLeast)));
}

// The unit that brings a row's largest to 2^kDsStart, from it and the present unit; not
// below `least`.
__device__ __forceinline__ int ds_unit(float most, int unit, int least) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
    return max(unit + e - kDsStart, least);
}

template <int N>
__device__ __forceinline__ void scale_sums(f32x16 (&x)[N], float f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] *= f;
}

// The unit of a row (its sums, and the largest scaled dS so far) where exponents go row by
// row: `most` is the exponent of the lane's largest dS times 2^e.
template <int N>
__device__ __forceinline__ void raise_unit(int most, int& unit, float& run, f32x16 (&sums)[N]) {
    most = max(most, __shfl_xor(most, 32));  // the row's other half
    if (run > 0.0f) most = max(most, attn_exponent(run) + unit - kAttnUnit);
    int to = unit;
    const int reach = kAttnUnit + most - unit;
    if (most > kUnset && (reach >= kDsMost || reach < kDsLeast)) to = most + kAttnUnit - kDsStart;
    scale_sums(sums, attn_pow2(unit - to));
    unit = to;
    run = most > kUnset ? attn_pow2(kAttnUnit + most - unit) : 0.0f;
}

__device__ __forceinline__ float largest(const float (&x)[16]) {
    float m = fabsf(x[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) m = fmaxf(m, fabsf(x[r]));
    return m;
}

// The diagonals of a block of 32 queries x 8 keys: a row of LDS each, eight keys
// wide and four more floats, so that 16-byte reads of 16 rows meet all banks.
constexpr int kDiags = 39, kDiagRow = 12;

// Between LDS writes and reads of one wave's lanes: they execute in order.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 64 floats of a row array into LDS, by one wave.
__device__ __forceinline__ void load_row(const float* from, AttnLds* to, int lane) {
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

// dK, dV: a workgroup takes 128 keys of one key head, a wave 32 of them. Its rows
// of K stay in registers, those of V too up to 64 features; at 128 they are read
// from LDS (in registers they spilled, and a reload waits for the loads ahead).
// Q and dO come through LDS, two buffers of 64 rows (32 at 128 features, which
// leaves room for two workgroups a CU), for every query head of the group in
// turn, or for some of them where a group is spread over workgroups. Scores are
// Q·K^T here: a lane holds 16 queries of one key, as the operands of
// dV^T = dO^T·P and dK^T = Q^T·dS need them. One sequence of 16384, 32 heads over 8
// of 128, bfloat16, causal: 5.0 ms, 0.88 PFLOP/s in its four products; the 512
// registers of a SIMD's lane hold two waves, too few to keep the matrix cores busy
// while both compute weights.
//
// ROWS: the form for workgroups that meet an uneven tile, exponents row by row; the other
// form leaves them to it. Two kernels, as one would keep registers for both and spill;
// where there are none the second reads a flag, 4.6 us with its launch.
template <bool SPLIT, int DB, bool BIAS, bool ROWS>
__global__ __launch_bounds__(kAttnThreads, DB * (SPLIT ? 2 : 1) <= 4 ? 2 : 1) void
attn_dkv_kernel(const AttnArgs g) {
    using T = AttnTile<DB>;
    constexpr int kPlanes = SPLIT ? 2 : 1, kTile = kPlanes * T::kPlane, KS = 2 * DB;
    constexpr int kLogDp = DB == 1 ? 5 : DB == 2 ? 6 : 7;
    constexpr bool kVInLds = DB == 4;
    constexpr int kRows = kVInLds ? 32 : 64;             // queries of a stage
    constexpr int kPart = kRows * T::kRowBytes;          // bytes of a plane of them
    constexpr int kBytes = kPlanes * kPart;
    constexpr int kRing = 2 * kBytes + (BIAS ? 768 : 512);
    __shared__ __align__(16) unsigned char ring0[kRing];
    __shared__ __align__(16) unsigned char ring1[kRing];
    __shared__ __align__(16) unsigned char values[kVInLds ? 2 * kTile : 16];
    // the last fragments of K, where registers would spill: each lane its own
    constexpr int kSpare = !kVInLds || SPLIT ? 0 : 3;
    __shared__ f16x8 spare[kSpare ? 4 * kSpare : 1][64];
    extern __shared__ float bias_row[];

    if (ROWS && attn_scalar(g.uneven) == 0) return;
    const int t = threadIdx.x, lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    // the query heads of the group that this part of it takes: rep from head0 on
    const int rep = g.heads / g.kv_heads / g.dkv_parts;
    const uint32_t u = blockIdx.x / g.kv_heads;
    const int kvh = blockIdx.x % g.kv_heads, part = u % g.dkv_parts;
    const int head0 = (kvh * g.dkv_parts + part) * rep;
    int sid, tile;
    if (!attn_entry(g.plan, u / g.dkv_parts, g.tiles, true, sid, tile)) return;
    const AttnSeq seq = attn_seq(g.plan, sid);
    const int shift = seq.nk - seq.nq;
    const int key0 = tile * 128 + 32 * wv, key = key0 + (lane & 31);

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int fb = 0; fb < DB; ++fb)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[fb][r] = dv[fb][r] = 0.0f;
    // dV in units of 2^(co - 28), dK of 2^(cq - 28), row by row: the largest exponent of
    // dO's tiles that the row's key is seen by, and dS's unit
    int co = kUnset, cq = kUnset;

    // stages of queries, from the first that sees a key of the workgroup
    const int first = g.causal ? max(0, tile * 128 - shift) / kRows : 0;
    const int n_q = (seq.nq + kRows - 1) / kRows;
    const int nt = tile * 128 < seq.nk && first < n_q ? n_q - first : 0;

    if (nt > 0) {
        const int64_t q_tile0 = seq.pq / 64;
        auto issue = [&](AttnLds* to, int hr, int qt) __attribute__((always_inline)) {
            const int head = head0 + hr, row = (first + qt) * kRows;
            const int64_t tq = q_tile0 + row / 64;
            const int64_t at = tq * kTile + (row & 63) * T::kRowBytes;
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) {
                attn_stage<kPart>(g.q.p + head * g.q.sh + at + p * T::kPlane, to + p * kPart, wv,
                                  lane);
                attn_stage<kPart>(g.dout.p + head * g.dout.sh + at + p * T::kPlane,
                                  to + kBytes + p * kPart, wv, lane);
            }
            // the whole tile's 64 rows each, of which a stage of 32 uses its half
            if (wv == 0) load_row(g.lse + head * g.lse_sh + tq * 64, to + 2 * kBytes, lane);
            if (wv == 1) load_row(g.delta + head * g.lse_sh + tq * 64, to + 2 * kBytes + 256, lane);
            if (BIAS && wv == 2)
                load_row(g.inv + head * g.lse_sh + tq * 64, to + 2 * kBytes + 512, lane);
        };
        issue((AttnLds*)ring0, 0, 0);
        const AttnReads<SPLIT, DB> rd(lane);
        // a tile of 64 rows, and a stage's
        auto row_of = [&](const unsigned char* buf, int b, int ks) __attribute__((always_inline)) {
            return rd.template along<kPart>(buf, b, ks);
        };

        const bool live = key0 < seq.nk;
        const int k_row = seq.pk + (live ? key0 : 0);
        AttnPair<SPLIT> kf[KS - kSpare], vf[kVInLds ? 1 : KS];
        {
            const int64_t at = static_cast<int64_t>(k_row / 64) * kTile;
            const unsigned char* ka =
                reinterpret_cast<const unsigned char*>(g.k.p + kvh * g.k.sh + at);
            const unsigned char* va =
                reinterpret_cast<const unsigned char*>(g.v.p + kvh * g.v.sh + at);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const AttnPair<SPLIT> x = rd.along(ka, (k_row >> 5) & 1, ks);
                if (ks < KS - kSpare) kf[ks < KS - kSpare ? ks : 0] = x;
                else spare[kSpare * wv + ks - (KS - kSpare)][lane] = x.f[0];
                if constexpr (!kVInLds) vf[ks] = rd.along(va, (k_row >> 5) & 1, ks);
            }
            if constexpr (kVInLds) {
                // the second of the workgroup's two tiles is there if a key of it is
                const char* from = g.v.p + kvh * g.v.sh + (seq.pk / 64 + 2 * tile) * int64_t{kTile};
                attn_stage<kTile>(from, (AttnLds*)values, wv, lane);
                if (tile * 128 + 64 < seq.nk)
                    attn_stage<kTile>(from + kTile, (AttnLds*)values + kTile, wv, lane);
            }
        }
        {
            // of all the tiles that the workgroup meets
            const int64_t k0 = seq.pk / 64 + 2 * tile;
            const int64_t k1 = k0 + (min(seq.nk - tile * 128, 128) + 63) / 64;
            const int64_t q0 = q_tile0 + first * kRows / 64, q1 = q_tile0 + (seq.nq + 63) / 64;
            int flags = attn_flags(g.k, kvh, k0, k1, lane) | attn_flags(g.v, kvh, k0, k1, lane);
            for (int h = head0; h < head0 + rep; ++h)
                flags |= attn_flags(g.q, h, q0, q1, lane) | attn_flags(g.dout, h, q0, q1, lane) |
                         attn_more_flags(g.q, h, q0, q1, lane) |
                         attn_more_flags(g.dout, h, q0, q1, lane);
            if (attn_uneven(flags) != ROWS) {
                if (!ROWS && t == 0) *g.uneven = 1;
                __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no loads into LDS outlive the workgroup
                return;
            }
        }
        const unsigned char* const my_v = values + (wv >> 1) * kTile;
        const int even_ke = attn_exp(g.k, kvh, k_row), even_ve = attn_exp(g.v, kvh, k_row);
        float run = 0.0f;  // the largest scaled |dS| of the lane's key so far
        // of the stage that they were set for: weights are times 2^unit, dS times 2^14 and the
        // row's unit is weight · beta · (dP - delta)
        float unit = 0.0f, beta = 0.0f;
        int set_oe = kUnset, set_qe = kUnset, set_b = kUnset;
        const int md = BIAS ? g.bias.max_distance : 0;

        auto compute = [&](const unsigned char* buf, int hr, int q_first)
            __attribute__((always_inline)) {
            const int head = head0 + hr, row0 = seq.pq + q_first;
            const int ke = ROWS ? *g.k.row(kvh, k_row + (lane & 31)) : even_ke;
            const int ve = ROWS ? *g.v.row(kvh, k_row + (lane & 31)) : even_ve;
            const int qe = attn_exp(g.q, head, row0), oe = attn_exp(g.dout, head, row0);
            const int de = attn_scalar(g.dexps + head * g.q.exps_sh + (row0 >> 6));
            const float c = ldexpf(g.scale2, min(qe + ke - 2 * kAttnUnit, 126));
            const float alpha = attn_pow2(oe + ve - 2 * kAttnUnit);
            const int b = ds_exponent(oe, ve, de, kLogDp);
            // the lane's key is seen by rows [from, to) of a block
            auto seen_from = [&](int q0) { return g.causal ? max(key - shift - q0, 0) : 0; };
            auto seen_to = [&](int q0) { return key < seq.nk ? min(seq.nq - q0, 32) : 0; };
            // A row that sees one key alone, the sequence's first, has weight 1 there and dS 0,
            // not what roundings leave of dP - delta (what is not finite stays so).
            auto single_key = [&](int k) {
                return seq.nk == 1 || (g.causal && k == 0);
            };
            auto only_key = [&](float* x, int r0, int q0) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (seq.nk == 1 || (key == 0 && q0 + attn_row(r0 + i, lane) + shift == 0))
                        x[i] *= 0.0f;
            };
            auto move = [&](int to) __attribute__((always_inline)) {  // dK's unit
                const float f = attn_pow2(cq - to);
                scale_sums(dk, f);
                run *= f;
                cq = to;
            };
#pragma unroll
            for (int qb = 0; qb < kRows / 32; ++qb) {
                const int q0 = q_first + 32 * qb;
                if (q0 >= seq.nq || (g.causal && q0 + 31 + shift < key0)) continue;
                const bool masked = q0 + 31 >= seq.nq || key0 + 31 >= seq.nk ||
                                    (g.causal && q0 + shift < key0 + 31);
                f32x16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
                attn_pipeline<SPLIT, 2 * KS, kAttnAhead<SPLIT>>(
                    [&](auto i) __attribute__((always_inline)) {
                        return row_of(i.value % 2 ? buf + kBytes : buf, qb, i.value / 2);
                    },
                    [&](auto i, const AttnPair<SPLIT>& x) __attribute__((always_inline)) {
                        constexpr int ks = i.value / 2;
                        if constexpr (i.value % 2 == 0) {
                            AttnPair<SPLIT> k = kf[ks < KS - kSpare ? ks : 0];
                            if constexpr (ks >= KS - kSpare)
                                k.f[0] = spare[kSpare * wv + ks - (KS - kSpare)][lane];
                            s = attn_dot<SPLIT>(x, k, s);
                        } else {
                            dp = attn_dot<SPLIT>(x, kVInLds ? rd.along(my_v, wv & 1, ks)
                                                            : vf[kVInLds ? 0 : ks], dp);
                        }
                    });
                const float* lse =
                    reinterpret_cast<const float*>(buf + 2 * kBytes) + (q0 & 63);
                const float* delta = lse + 64;
                // the bias of the block's first query and this key; far: the same for all
                const int lo_d = q0 + shift - key0 - 31;
                const bool far = BIAS && (lo_d >= md || lo_d + 62 <= -md);
                const float flat = BIAS ? bias_row[kAttnFar + (lo_d >= md ? 2 * md : 0)] : 0.0f;
                const float* const near_at =
                    BIAS ? bias_row + md + kAttnFar + (far ? 0 : q0 + shift - key) +
                               4 * (lane >> 5)
                         : nullptr;
                if (!ROWS && (masked || oe != set_oe || qe != set_qe || b > set_b)) {
                    const bool sees = !masked || seen_from(q0) < seen_to(q0);
                    if (__builtin_amdgcn_ballot_w64(sees & (oe > co)) != 0) {
                        const int to = sees ? max(co, oe) : co;
                        scale_sums(dv, attn_pow2(co - to));
                        co = to;
                    }
                    const int u = kAttnUnit + max(oe - co, -60);
                    const int to = sees ? max(cq, qe + kAttnUnit - u + b - kDsReach) : cq;
                    if (__builtin_amdgcn_ballot_w64(to != cq) != 0) move(to + (to != cq ? 14 : 0));
                    unit = static_cast<float>(u);
                    beta = attn_pow2(qe + kAttnUnit - u - cq);
                    set_oe = masked ? kUnset : oe;  // other rows are seen in the next one
                    set_qe = qe;
                    set_b = b;
                }
                AttnPair<SPLIT> wp[1][2], wd[1][2];
                float ds[16];
                if constexpr (ROWS) {
                    const int lo = seen_from(q0), hi = seen_to(q0);
                    const int64_t at_row = row0 + 32 * qb + 4 * (lane >> 5);
                    float p[16];
                    int most_o = kUnset, most = kUnset;  // of what the key is seen by
                    uint32_t qx[4], ox[4];
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        qx[r4] = attn_four_rows(g.q.row(head, at_row + 8 * r4));
                        ox[r4] = attn_four_rows(g.dout.row(head, at_row + 8 * r4));
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int row = attn_row(r, lane);
                        const int qr = attn_one_of(qx[r / 4], r % 4);
                        const int dr = attn_one_of(ox[r / 4], r % 4);
                        float x = ldexpf(s[r] * g.scale2, qr + ke - 2 * kAttnUnit);
                        if constexpr (BIAS)
                            x += far ? flat : near_at[8 * (r / 4) + r % 4];
                        p[r] = attn_exp2(x - lse[row]);
                        if constexpr (BIAS) p[r] *= lse[128 + row];
                        ds[r] = p[r] * (ldexpf(dp[r], dr + ve - 2 * kAttnUnit) - delta[row]);
                        const bool see = row >= lo && row < hi;
                        p[r] = see ? p[r] : 0.0f;
                        ds[r] = see ? ds[r] : 0.0f;
                        if (p[r] != 0.0f) most_o = max(most_o, dr);
                    }
                    if (single_key(key0)) {
                        only_key(ds, 0, q0);
                        only_key(ds + 8, 8, q0);
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (ds[r] != 0.0f)
                            most = max(most,
                                       attn_exponent(ds[r]) + attn_one_of(qx[r / 4], r % 4));
                    most_o = max(max(most_o, __shfl_xor(most_o, 32)), co);
                    scale_sums(dv, attn_pow2(co - most_o));
                    co = most_o;
                    raise_unit(most, cq, run, dk);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        p[r] = ldexpf(p[r], kAttnUnit + attn_one_of(ox[r / 4], r % 4) - co);
                        ds[r] = ldexpf(ds[r], kAttnUnit + attn_one_of(qx[r / 4], r % 4) - cq);
                    }
                    wp[0][0] = attn_operand<SPLIT>(p);
                    wp[0][1] = attn_operand<SPLIT>(p + 8);
                }
#pragma unroll
                for (int half = 0; half < (ROWS ? 0 : 2); ++half) {
                    float p[8];
#pragma unroll
                    for (int r4 = 0; r4 < 2; ++r4) {
                        const int at = 16 * half + 8 * r4, row = at + 4 * (lane >> 5);
                        const f32x4 z = *reinterpret_cast<const f32x4*>(lse + row);
                        const f32x4 d = *reinterpret_cast<const f32x4*>(delta + row);
                        f32x4 inv = z;
                        if constexpr (BIAS) inv = *reinterpret_cast<const f32x4*>(lse + 128 + row);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = 4 * r4 + j, r = 8 * half + i;
                            // with a bias, rounded as in the forward: it may swallow the score
                            if constexpr (BIAS)
                                p[i] = attn_exp2(__builtin_fmaf(s[r], c,
                                                                far ? flat : near_at[at + j]) -
                                                 z[j] + unit) * inv[j];
                            else p[i] = attn_exp2(__builtin_fmaf(s[r], c, unit - z[j]));
                            ds[r] = p[i] * beta * __builtin_fmaf(dp[r], alpha, -d[j]);
                        }
                    }
                    if (masked) {
                        const int lo = seen_from(q0), hi = seen_to(q0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int row = attn_row(8 * half + i, lane);
                            const bool see = row >= lo && row < hi;
                            p[i] = see ? p[i] : 0.0f;
                            ds[8 * half + i] = see ? ds[8 * half + i] : 0.0f;
                        }
                        if (single_key(key0)) only_key(ds + 8 * half, 8 * half, q0);
                    }
                    wp[0][half] = attn_operand<SPLIT>(p);
                }
                if constexpr (!ROWS) run = fmaxf(run, largest(ds));
                if (!ROWS && __builtin_amdgcn_ballot_w64(ds_out(run)) != 0) {
                    run = fmaxf(run, __shfl_xor(run, 32));  // the key's other half
                    const bool out = ds_out(run);
                    const int u = static_cast<int>(unit);
                    const int to =
                        out ? ds_unit(run, cq, qe + kAttnUnit - u + b - kDsReach) : cq;
                    const float f = attn_pow2(cq - to);
                    move(to);
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] *= f;
                    // where the bound kept it from rising it is not tried again
                    if (out) run = fmaxf(run, static_cast<float>(1 << kDsLeast));
                    beta *= f;
                    set_b = b;
                }
                wd[0][0] = attn_operand<SPLIT>(ds);
                wd[0][1] = attn_operand<SPLIT>(ds + 8);
                attn_accumulate<SPLIT, DB, 1, kPart>(rd, buf + kBytes, qb, wp, dv);
                attn_accumulate<SPLIT, DB, 1, kPart>(rd, buf, qb, wd, dk);
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
            if (hr < rep) issue((AttnLds*)next, hr, qt);
            if (BIAS && i == 0) {  // a head's first stage
                attn_bias_row(g.bias, head0 + h, bias_row);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            if (live) compute(cur, h, (first + i) * kRows);
        };
        int left = rep * nt;
        for (; left >= 2; left -= 2) {
            stage(ring0, ring1);
            stage(ring1, ring0);
        }
        if (left) stage(ring0, ring1);
    }

    if (key >= seq.ek || (ROWS && nt == 0)) return;
    const float fk = ldexpf(g.scale, cq - 2 * kAttnUnit), fv = attn_pow2(co - 2 * kAttnUnit);
    const bool zero = key >= seq.nk || nt == 0;
    if (g.dkv_parts > 1 && key < seq.nk) {
        const int64_t row = static_cast<int64_t>(kvh) * g.dkv_rows + seq.pk + key;
        const int64_t step = static_cast<int64_t>(g.kv_heads) * g.dkv_rows;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float* const at = g.dkv_part + ((2 * part + which) * step + row) * T::DP;
#pragma unroll
            for (int fb = 0; fb < DB; ++fb)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    f32x4 x;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[j] = zero ? 0.0f
                                    : (which ? dv[fb] : dk[fb])[4 * r4 + j] * (which ? fv : fk);
                    *reinterpret_cast<f32x4*>(at + 32 * fb + 8 * r4 + 4 * (lane >> 5)) = x;
                }
        }
        return;
    }
    if (part != 0) return;  // the first part writes what no key stands behind
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
// Q and dO stay in registers; K and V come through LDS. The bias's gradient: a wave
// lays eight keys' dS out by diagonals in LDS, sums each in one lane and adds it to
// the wave's own bin of that distance, so the sums need no atomicity and repeat.
// (Float atomics on LDS took some 260 cycles an instruction: the whole kernel 137
// us, without them 65, at 16 x 512 tokens, 12 heads of 64, float32.) One sequence of
// 16384, 32 heads over 8 of 128, bfloat16, causal: 3.0 ms, 1.10 PFLOP/s in its three
// products, bound by the matrix cores and the softmax's instructions between them.
template <bool SPLIT, int DB, bool BIAS>
__global__ __launch_bounds__(kAttnThreads, DB * (SPLIT ? 2 : 1) <= 4 ? 2 : 1) void
attn_dq_kernel(const AttnArgs g) {
    using T = AttnTile<DB>;
    constexpr int kBytes = (SPLIT ? 2 : 1) * T::kPlane, KS = 2 * DB;
    constexpr int kLogDp = DB == 1 ? 5 : DB == 2 ? 6 : 7;
    __shared__ __align__(16) unsigned char ring0[2 * kBytes];
    __shared__ __align__(16) unsigned char ring1[2 * kBytes];
    extern __shared__ __align__(16) float lds_floats[];

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
    float* const diag = lds_floats + (threadIdx.x >> 6) * kDiags * kDiagRow;
    float* const far = lds_floats + 4 * kDiags * kDiagRow;  // [wave][below, above]
    float* const bias_row = far + 8;
    float* const bins = bias_row + attn_bias_floats(md);  // [wave][distance]
    // Of a single key that a query sees the weight is 1 and dS 0, not what roundings leave of
    // dP - delta (what is not finite stays so).
    auto sees_one = [&]() { return seq.nk == 1 || (g.causal && q + shift == 0); };
    const int d_row = min(lane, kDiags - 1);
    float below = 0.0f, above = 0.0f;            // distances past the last bins
    if constexpr (BIAS) {
        attn_bias_row(g.bias, head, bias_row);
        for (int i = t; i < 4 * width; i += kAttnThreads) bins[i] = 0.0f;
        for (int i = lane; i < kDiags * kDiagRow; i += 64) diag[i] = 0.0f;
    }

    f32x16 dq[DB];
#pragma unroll
    for (int fb = 0; fb < DB; ++fb)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[fb][r] = 0.0f;
    int ck = kUnset;  // dQ in units of 2^(ck - 28), row by row
    float run = 0.0f;  // the largest scaled |dS| of the lane's query so far

    if (t1 > 0) {
        const int64_t k_tile = seq.pk / 64;
        auto issue = [&](AttnLds* to, int kt) __attribute__((always_inline)) {
            const int64_t at = (k_tile + kt) * kBytes;
            attn_stage<kBytes>(g.k.p + kvh * g.k.sh + at, to, wv, lane);
            attn_stage<kBytes>(g.v.p + kvh * g.v.sh + at, to + kBytes, wv, lane);
        };
        issue((AttnLds*)ring0, 0);
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
        const float inv = BIAS && mine ? g.inv[ri] : 0.0f;
        const float delta = mine ? g.delta[ri] : 0.0f;
        const int even_qe = attn_exp(g.q, head, q_row), even_oe = attn_exp(g.dout, head, q_row);
        const int de = attn_scalar(g.dexps + head * g.q.exps_sh + (q_row >> 6));

        int set_b = kUnset;  // the largest exponent, K's counted, that ck was looked at for
        auto move = [&](int to) __attribute__((always_inline)) {
            const float f = attn_pow2(ck - to);
            scale_sums(dq, f);
            run *= f;
            ck = to;
        };
        // ROWS: exponents row by row, as uneven tiles have them
        auto compute = [&](auto rows, const unsigned char* buf, int key_tile)
            __attribute__((always_inline)) {
            constexpr bool ROWS = decltype(rows)::value;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key0 = key_tile + 32 * kb;
                if (key0 >= seq.nk) return;
                if (g.causal && key0 > wave0 + 31 + shift) return;
                const bool masked =
                    key0 + 31 >= seq.nk || (g.causal && key0 + 31 > wave0 + shift);
                const int ke = attn_exp(g.k, kvh, seq.pk + key0);
                const int ve = attn_exp(g.v, kvh, seq.pk + key0);
                const int qe = ROWS ? *g.q.row(head, q_row + (lane & 31)) : even_qe;
                const int oe = ROWS ? *g.dout.row(head, q_row + (lane & 31)) : even_oe;
                const float c = ldexpf(g.scale2, min(qe + ke - 2 * kAttnUnit, 126));
                const int b = ds_exponent(oe, ve, de, kLogDp);
                if (!ROWS && ke + b > set_b) {
                    const int to = max(ck, ke + b - kDsReach);
                    if (__builtin_amdgcn_ballot_w64(to != ck) != 0) move(to + (to != ck ? 14 : 0));
                    set_b = ke + b;
                }
                // dS times 2^x: dP and delta are; in the weights' exponent x would round it
                const int x = kAttnUnit + ke - ck;
                const float alpha = attn_pow2(x + oe + ve - 2 * kAttnUnit);
                const float db = delta * attn_pow2(x);
                // The matrix cores' sums err downwards, which the bias's gradient, a sum
                // of many dS that cancel, would collect: its small products go apart.
                constexpr bool kApart = SPLIT && BIAS;
                f32x16 s, dp, small;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = dp[r] = small[r] = 0.0f;
                attn_pipeline<SPLIT, 2 * KS, kAttnAhead<SPLIT>>(
                    [&](auto i) __attribute__((always_inline)) {
                        return rd.along(i.value % 2 ? buf + kBytes : buf, kb, i.value / 2);
                    },
                    [&](auto i, const AttnPair<SPLIT>& x) __attribute__((always_inline)) {
                        if constexpr (i.value % 2 == 0)
                            s = attn_dot<SPLIT>(x, qf[i.value / 2], s);
                        else if constexpr (kApart)
                            dp = attn_dot_apart(x, of[i.value / 2], dp, small);
                        else dp = attn_dot<SPLIT>(x, of[i.value / 2], dp);
                    });
                if constexpr (kApart) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) dp[r] += small[r];
                }
                const int lim = (g.causal ? min(seq.nk - 1, q + shift) : seq.nk - 1) - key0;
                const int away = q + shift - key0;
                bool near = false;
                float flat = 0.0f;
                if constexpr (BIAS) {
                    const int lo = wave0 + shift - key0 - 31, hi = lo + 62;
                    near = lo < md && hi > -md;
                    flat = bias_row[kAttnFar + (lo >= md ? 2 * md : 0)];
                }
                const float* const near_at = BIAS ? bias_row + md + kAttnFar +
                                                        (near ? away - 4 * (lane >> 5) : 27) - 27
                                                  : nullptr;
                float ds[16];
                uint32_t kx[4], vx[4];
                if constexpr (ROWS) {
                    const int64_t at = seq.pk + key0 + 4 * (lane >> 5);
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        kx[r4] = attn_four_rows(g.k.row(kvh, at + 8 * r4));
                        vx[r4] = attn_four_rows(g.v.row(kvh, at + 8 * r4));
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float p;
                    if constexpr (ROWS) {
                        float x = ldexpf(s[r] * g.scale2,
                                         qe + attn_one_of(kx[r / 4], r % 4) - 2 * kAttnUnit);
                        if constexpr (BIAS)
                            x += near ? near_at[27 - 8 * (r >> 2) - (r & 3)] : flat;
                        p = attn_exp2(x - lse);
                        if constexpr (BIAS) p *= inv;
                        ds[r] = p * (ldexpf(dp[r], oe + attn_one_of(vx[r / 4], r % 4) -
                                                       2 * kAttnUnit) - delta);
                        continue;
                    }
                    if constexpr (BIAS)
                        p = attn_exp2(__builtin_fmaf(s[r], c,
                                                     near ? near_at[27 - 8 * (r >> 2) - (r & 3)]
                                                          : flat) - lse) * inv;
                    else p = attn_exp2(__builtin_fmaf(s[r], c, -lse));
                    ds[r] = p * __builtin_fmaf(dp[r], alpha, -db);
                }
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        ds[r] = attn_row(r, lane) <= lim ? ds[r] : 0.0f;
                }
                if (BIAS && key0 == 0 && sees_one()) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] *= 0.0f;
                }
                if constexpr (BIAS) {
                    if (near) {
                        // eight keys at a time: lane d sums the diagonal of distance
                        // d - 7 from the first key's of the first query
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int k = 4 * (lane >> 5) + j;
                                diag[((lane & 31) - k + 7) * kDiagRow + k] =
                                    ROWS ? ds[4 * r4 + j] : ldexpf(ds[4 * r4 + j], -x);
                            }
                            wave_lds_fence();
                            const f32x4* const at =
                                reinterpret_cast<const f32x4*>(diag + d_row * kDiagRow);
                            const f32x4 lo = at[0], hi = at[1];
                            float y = ((lo[0] + lo[1]) + (lo[2] + lo[3])) +
                                      ((hi[0] + hi[1]) + (hi[2] + hi[3]));
                            y = lane < kDiags ? y : 0.0f;
                            const int d = wave0 + shift - key0 - 8 * r4 + d_row - 7;
                            if (d >= md) above += y;
                            else if (d <= -md) below += y;
                            else if (lane < kDiags) bins[wv * width + md + d] += y;
                            wave_lds_fence();
                        }
                    } else {
                        float y = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) y += ds[r];
                        if constexpr (!ROWS) y = ldexpf(y, -x);
                        if (away >= md) above += y;
                        else below += y;
                    }
                }
                if constexpr (ROWS) {
                    int most = kUnset;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (ds[r] != 0.0f)
                            most = max(most, attn_exponent(ds[r]) + attn_one_of(kx[r / 4], r % 4));
                    raise_unit(most, ck, run, dq);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        ds[r] = ldexpf(ds[r], kAttnUnit + attn_one_of(kx[r / 4], r % 4) - ck);
                } else {
                    run = fmaxf(run, largest(ds));
                }
                if (!ROWS && __builtin_amdgcn_ballot_w64(ds_out(run)) != 0) {
                    run = fmaxf(run, __shfl_xor(run, 32));  // the query's other half
                    const bool out = ds_out(run);
                    const int to = out ? ds_unit(run, ck, ke + b - kDsReach) : ck;
                    const float f = attn_pow2(ck - to);
                    move(to);
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] *= f;
                    if (out) run = fmaxf(run, static_cast<float>(1 << kDsLeast));
                    set_b = ke + b;
                }
                const AttnPair<SPLIT> w[1][2] = {
                    {attn_operand<SPLIT>(ds), attn_operand<SPLIT>(ds + 8)}};
                attn_accumulate<SPLIT, DB, 1>(rd, buf, kb, w, dq);
            }
        };
        auto stage = [&](auto rows, const unsigned char* cur, unsigned char* next, int kt)
            __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(wait_vm(0));
            asm volatile("s_barrier" ::: "memory");
            if (kt + 1 < t1) issue((AttnLds*)next, kt + 1);
            if (wave0 < seq.nq) compute(rows, cur, kt * kAttnRows);
        };
        auto all = [&](auto rows) __attribute__((always_inline)) {
            int kt = 0;
            for (; kt + 2 <= t1; kt += 2) {
                stage(rows, ring0, ring1, kt);
                stage(rows, ring1, ring0, kt + 1);
            }
            if (kt < t1) stage(rows, ring0, ring1, kt);
        };
        // of all the tiles that the workgroup meets
        const int64_t q0 = (seq.pq + rows0) / 64, q1 = q0 + (min(seq.nq - rows0, 128) + 63) / 64;
        if (attn_uneven(attn_flags(g.q, head, q0, q1, lane) |
                        attn_flags(g.dout, head, q0, q1, lane) |
                        attn_flags(g.k, kvh, k_tile, k_tile + t1, lane) |
                        attn_flags(g.v, kvh, k_tile, k_tile + t1, lane) |
                        attn_more_flags(g.k, kvh, k_tile, k_tile + t1, lane) |
                        attn_more_flags(g.v, kvh, k_tile, k_tile + t1, lane)))
            all(std::true_type{});
        else all(std::false_type{});
    }

    if (q < seq.eq && g.dq.p != nullptr) {
        const bool zero = q >= seq.nq || t1 == 0;
        const float f = zero         ? 1.0f
                        : sees_one() ? 0.0f
                                     : ldexpf(g.scale, ck - 2 * kAttnUnit);
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
            for (int j = 0; j < 4; ++j) y += bins[j * width + i];
            for (int j = 0; j < 4; ++j) y += i == 0 ? far[2 * j] : i == 2 * md ? far[2 * j + 1] : 0.0f;
            out[i] = y;
            if (slots > 1) out[width + i] = 0.0f;
        }
    }
}

// Sums the parts of dk and dv: half a wave a row of one of them, four features a
// lane.
__global__ __launch_bounds__(kAttnThreads) void attn_dkv_join_kernel(const AttnArgs g, int dp) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int kvh = blockIdx.y, which = (threadIdx.x >> 5) & 1, f = 4 * (threadIdx.x & 31);
    const AttnRow r = attn_row_of(g.plan, true, row);
    if (!r.any || r.row >= r.seq.nk || f >= g.dim) return;
    const int64_t step = static_cast<int64_t>(g.kv_heads) * g.dkv_rows;
    const float* from = g.dkv_part + (which * step + kvh * g.dkv_rows + row) * dp + f;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int p = 0; p < g.dkv_parts; ++p) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(from + 2 * p * step * dp);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += y[j];
    }
    const AttnIo& io = which ? g.dv : g.dk;
    const int64_t to = r.sid * io.sb + (r.seq.k0 + r.row) * io.sr + kvh * io.sh;
    if (io.sd == 1 && g.vec_kv) {
        if (g.dtype == SLK_F32) F32::store4(io.p, to + f, x);
        else BF16::store4(io.p, to + f, x);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (f + j >= g.dim) return;
        if (g.dtype == SLK_F32) F32::store(io.p, to + (f + j) * io.sd, x[j]);
        else BF16::store(io.p, to + (f + j) * io.sd, x[j]);
    }
}

// The bias's gradient from the workgroups' bins, in their order: a workgroup a
// head, four threads a distance (a quarter of the bins each), then a thread a
// bucket.
__global__ __launch_bounds__(1024) void attn_dbias_kernel(const AttnArgs g, void* dbias) {
    constexpr int kMost = 2 * SLK_ATTN_MAX_DISTANCE + 1;
    __shared__ float quarter[4][kMost];
    __shared__ float per[kMost];
    const int head = blockIdx.x, md = g.bias.max_distance, width = 2 * md + 1;
    const int64_t rows = g.plan.seqs != nullptr ? g.plan.count[1] : g.plan.batch * g.plan.pad_t;
    const int64_t slots = rows / kAttnRows;
    const float* from = g.dbias_part + head * g.dbias_slots * width;
    const int part = threadIdx.x >> 8;
    const int64_t s0 = slots * part / 4, s1 = slots * (part + 1) / 4;
    for (int i = threadIdx.x & 255; i < width; i += 256) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = 0.0f;
        int64_t s = s0;
        for (; s + 8 <= s1; s += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] += from[(s + j) * width + i];
        }
        for (; s < s1; ++s) y[0] += from[s * width + i];
        quarter[part][i] = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += 1024)
        per[i] = (quarter[0][i] + quarter[1][i]) + (quarter[2][i] + quarter[3][i]);
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
        k_entries * g.kv_heads * g.dkv_parts > max_groups(kAttnThreads))
        return fail(SLK_EINVAL, "attention_backward: too many tiles");
    if (want_kv) {
        AttnArgs a = g;
        a.plan = kplan;
        a.tiles = k_tiles;
        const dim3 grid(static_cast<unsigned>(k_entries * g.kv_heads * g.dkv_parts));
        const size_t lds = BIAS ? attn_bias_floats(g.bias.max_distance) * sizeof(float) : 0;
        hipLaunchKernelGGL((attn_dkv_kernel<SPLIT, DB, BIAS, false>), grid, dim3(kAttnThreads), lds,
                           st, a);
        hipLaunchKernelGGL((attn_dkv_kernel<SPLIT, DB, BIAS, true>), grid, dim3(kAttnThreads), lds,
                           st, a);
        const int rc = check_launch("attention_backward: dk, dv");
        if (rc != SLK_OK) return rc;
        if (g.dkv_parts > 1) {
            hipLaunchKernelGGL(attn_dkv_join_kernel,
                               dim3(static_cast<unsigned>(g.dkv_rows / 4), g.kv_heads),
                               dim3(kAttnThreads), 0, st, a, 32 * DB);
            const int rj = check_launch("attention_backward: join");
            if (rj != SLK_OK) return rj;
        }
    }
    if (want_q) {
        hipLaunchKernelGGL((attn_dq_kernel<SPLIT, DB, BIAS>),
                           dim3(static_cast<unsigned>(q_entries * g.heads)), dim3(kAttnThreads),
                           BIAS ? (attn_bias_floats(g.bias.max_distance) + 4 * width + 8 +
                                   4 * kDiags * kDiagRow) * sizeof(float)
                                : 0,
                           st, g);
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
