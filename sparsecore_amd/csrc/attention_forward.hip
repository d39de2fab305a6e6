// slk_attention_forward's kernel.
#include "attention.hpp"
#include "elem.hpp"

namespace slk {

namespace {

// Largest growth (in log 2) of a row's maximum that is left in its exponentials
// before the row is rescaled, and where packed weights start: below 2^15 in all.
constexpr float kGrowth = 8.0f;
constexpr int kWeightUnit = 7;

// A workgroup takes 128·QB queries of one head, a wave 32·QB of them; keys and
// values come through LDS, 64 at a time, two buffers, one barrier a tile. The
// scores of 32 keys are computed as K·Q^T, so that a lane holds 16 of them for
// one query (the other 16 are 32 lanes away): the softmax's maximum and sum are
// the lane's own, and its weights are the operand of O^T = V^T·P^T as they are.
// The row's maximum is only raised when a new one is more than 2^8 times above.
template <bool SPLIT, int DB, int QB, bool BIAS>
__global__ __launch_bounds__(kAttnThreads, DB * QB * (SPLIT ? 2 : 1) <= 4 ? 2 : 1) void
attn_forward_kernel(const AttnArgs g) {
    using T = AttnTile<DB>;
    constexpr int kPlanes = SPLIT ? 2 : 1, kBytes = kPlanes * T::kPlane, KS = 2 * DB;
    __shared__ __align__(16) unsigned char ring0[2 * kBytes];
    __shared__ __align__(16) unsigned char ring1[2 * kBytes];
    extern __shared__ float bias_row[];

    const int t = threadIdx.x, lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t rep = g.heads / g.kv_heads;
    const uint32_t block = blockIdx.x;
    const uint32_t kvh = block % g.kv_heads, u0 = block / g.kv_heads;
    const uint32_t hg = u0 % rep, u1 = u0 / rep;
    const int split = static_cast<int>(u1 % g.splits);
    const int head = static_cast<int>(kvh * rep + hg);
    int sid, tile;
    if (!attn_entry(g.plan, u1 / g.splits, g.tiles, false, sid, tile)) return;
    const AttnSeq seq = attn_seq(g.plan, sid);
    const int rows0 = tile * 128 * QB, shift = seq.nk - seq.nq;
    const int wave0 = rows0 + 32 * QB * wv;
    const int q = wave0 + (lane & 31);  // + 32 qb

    // keys that the workgroup's queries see, and this part's share of their tiles
    const int last_q = min(rows0 + 128 * QB, seq.nq) - 1;
    const int seen = last_q < rows0 ? 0 : g.causal ? min(seq.nk, last_q + shift + 1) : seq.nk;
    const int n_tiles = seen <= 0 ? 0 : (seen + kAttnRows - 1) / kAttnRows;
    const int per = (n_tiles + g.splits - 1) / g.splits;
    const int t0 = min(split * per, n_tiles), t1 = min(t0 + per, n_tiles);

    float m[QB], l[QB];
    f32x16 o[DB][QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        m[qb] = -INFINITY;
        l[qb] = 0.0f;
#pragma unroll
        for (int fb = 0; fb < DB; ++fb)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[fb][qb][r] = 0.0f;
    }
    int vmax = -200;  // exponent that the accumulated values are in units of

    if (t0 < t1) {
        const int krows = g.k.packed ? (seq.nk + kAttnRows - 1) / kAttnRows * kAttnRows : seq.nk;
        const AttnLoads<SPLIT, DB> lk(g.k, g.k.rows(sid, seq.k0, seq.pk, kvh), krows, wv, lane);
        const AttnLoads<SPLIT, DB> lv(g.v, g.v.rows(sid, seq.k0, seq.pk, kvh), krows, wv, lane);
        const AttnReads<SPLIT, DB> rd(lane);
        lk.issue(ring0, t0 * kAttnRows, wv);
        lv.issue(ring0 + kBytes, t0 * kAttnRows, wv);

        AttnPair<SPLIT> qf[QB][KS];
        int qe[QB];
        {
            const char* base = g.q.rows(sid, seq.q0, seq.pq, head);
            const int qrows =
                g.q.packed ? (seq.nq + kAttnRows - 1) / kAttnRows * kAttnRows : seq.nq;
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const int64_t row = min(q + 32 * qb, qrows - 1);
                const char* at = base + row * g.q.sr + 16 * (lane >> 5);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int p = 0; p < kPlanes; ++p)
                        qf[qb][ks].f[p] = *reinterpret_cast<const AttnFrag<SPLIT>*>(
                            at + 32 * ks + (p ? g.q.plane : 0));
                qe[qb] = 0;
                if constexpr (SPLIT)
                    qe[qb] = attn_exp(g.q, head,
                                      seq.pq + min(wave0 + 32 * qb, qrows - 32));
            }
        }
        if constexpr (SPLIT) {
            int e = -200;
            for (int i = seq.pk / 32 + 2 * t0 + lane; i < seq.pk / 32 + 2 * t1; i += 64)
                e = max(e, g.v.exps[kvh * g.v.exps_sh + i]);
#pragma unroll
            for (int x = 32; x > 0; x >>= 1) e = max(e, __shfl_xor(e, x));
            vmax = __builtin_amdgcn_readfirstlane(e);
        }
        if constexpr (BIAS) attn_bias_row(g.bias, g.heads, head, bias_row);
        const int md = BIAS ? g.bias.max_distance : 0;

        auto compute = [&](const unsigned char* buf, int key_tile) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key0 = key_tile + 32 * kb;
                // a wave's last query sees no key of this block, or there is none
                if (key0 >= seq.nk) return;
                if (g.causal && key0 > wave0 + 32 * QB - 1 + shift) return;
                const bool masked =
                    key0 + 31 >= seq.nk || (g.causal && key0 + 31 > wave0 + shift);
                f32x16 s[QB];
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[qb][r] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const AttnPair<SPLIT> kf = rd.along(buf, kb, ks);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb)
                        s[qb] = attn_dot<SPLIT>(kf, qf[qb][ks], s[qb]);
                }
                float unit = 0.0f, back = 1.0f;
                int ke = 0;
                if constexpr (SPLIT) {
                    ke = attn_exp(g.k, kvh, seq.pk + key0);
                    const int d = max(attn_exp(g.v, kvh, seq.pk + key0) - vmax, -60);
                    unit = static_cast<float>(kWeightUnit + d);
                    back = attn_pow2(-d);
                }
                AttnPair<SPLIT> w[QB][2];
                uint32_t bits[QB];
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) {
                    float c = g.scale2;
                    if constexpr (SPLIT) c = ldexpf(c, qe[qb] + ke - 2 * kAttnUnit);
                    const int at = q + 32 * qb;
                    // the last key that this query sees, from the block's first
                    const int lim =
                        (g.causal ? min(seq.nk - 1, at + shift) : seq.nk - 1) - key0;
                    bits[qb] = 0xffff;
                    if constexpr (BIAS) {
                        const int away = at + shift - key0;  // distance of the block's key 0
                        const int lo = wave0 + 32 * qb + shift - key0 - 31, hi = lo + 62;
                        if (lo >= md || hi <= -md) {
                            const float b = bias_row[lo >= md ? 2 * md : 0];
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[qb][r] = __builtin_fmaf(s[qb][r], c, b);
                        } else {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                s[qb][r] = __builtin_fmaf(
                                    s[qb][r], c,
                                    bias_row[md + attn_clamp(away - attn_row(r, lane), md)]);
                        }
                        c = 1.0f;
                    }
                    if (masked) {
                        bits[qb] = 0;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const bool see = attn_row(r, lane) <= lim;
                            s[qb][r] = see ? s[qb][r] : -INFINITY;
                            bits[qb] |= (see ? 1u : 0u) << r;
                        }
                        // the scores' factor may be 0: not on the masked ones
                        if constexpr (!BIAS) {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                s[qb][r] = (bits[qb] >> r) & 1 ? s[qb][r] * c : s[qb][r];
                            c = 1.0f;
                        }
                    }
                    float top = s[qb][0];
#pragma unroll
                    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[qb][r]);
                    top = fmaxf(top, __shfl_xor(top, 32)) * c;
                    if (__builtin_amdgcn_ballot_w64(top > m[qb] + kGrowth) != 0) {
                        const float up = fmaxf(m[qb], top);
                        const float a = up == -INFINITY ? 1.0f : attn_exp2(m[qb] - up);
                        m[qb] = up;
                        l[qb] *= a;
#pragma unroll
                        for (int fb = 0; fb < DB; ++fb)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[fb][qb][r] *= a;
                    }
                    const float ref = (m[qb] == -INFINITY ? 0.0f : m[qb]) - unit;
                    float sum = 0.0f;
                    float p[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        p[r] = attn_exp2(__builtin_fmaf(s[qb][r], c, -ref));
                        sum += p[r];
                    }
                    l[qb] = __builtin_fmaf(sum, back, l[qb]);
                    w[qb][0] = attn_operand<SPLIT>(p);
                    w[qb][1] = attn_operand<SPLIT>(p + 8);
                }
                attn_accumulate<SPLIT, DB, QB>(rd, buf + kBytes, kb, w, o, masked, bits);
            }
        };
        auto stage = [&](const unsigned char* cur, unsigned char* next, int kt) __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(wait_vm(0));
            asm volatile("s_barrier" ::: "memory");
            if (kt + 1 < t1) {
                lk.issue(next, (kt + 1) * kAttnRows, wv);
                lv.issue(next + kBytes, (kt + 1) * kAttnRows, wv);
            }
            if (wave0 < seq.nq) compute(cur, kt * kAttnRows);
        };
        int kt = t0;
        for (; kt + 2 <= t1; kt += 2) {
            stage(ring0, ring1, kt);
            stage(ring1, ring0, kt + 1);
        }
        if (kt < t1) stage(ring0, ring1, kt);
    }

    const float unit = SPLIT ? attn_pow2(vmax - kAttnUnit) : 1.0f;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        float sum = l[qb] + __shfl_xor(l[qb], 32);
        const int at = q + 32 * qb;
        if (g.splits > 1) {
            // the join's unit: what is not scaled by this part's own exponent
            if (at >= seq.nq) {
                // rows that are written but are no queries: zeros, by the first part
                if (split == 0 && at < seq.eq) {
                    const int64_t to = sid * g.out.sb + (seq.q0 + at) * g.out.sr + head * g.out.sh;
                    for (int f = lane >> 5; f < g.dim; f += 2) {
                        if (g.dtype == SLK_F32) F32::store(g.out.p, to + f * g.out.sd, 0.0f);
                        else BF16::store(g.out.p, to + f * g.out.sd, 0.0f);
                    }
                }
                continue;
            }
            const int64_t row = (static_cast<int64_t>(split) * g.heads + head) * g.part_rows +
                                seq.pq + at;
            if (lane < 32) {
                g.part_ml[2 * row] = m[qb];
                g.part_ml[2 * row + 1] = SPLIT ? sum * attn_pow2(-kWeightUnit) : sum;
            }
            const float f = SPLIT ? unit * attn_pow2(-kWeightUnit) : 1.0f;
#pragma unroll
            for (int fb = 0; fb < DB; ++fb)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    f32x4 x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = o[fb][qb][4 * r4 + j] * f;
                    *reinterpret_cast<f32x4*>(g.part + row * T::DP + 32 * fb + 8 * r4 +
                                              4 * (lane >> 5)) = x;
                }
            continue;
        }
        if (g.lse != nullptr && lane < 32 && at < (seq.nq + kAttnRows - 1) / kAttnRows * kAttnRows) {
            const float z = SPLIT ? sum * attn_pow2(-kWeightUnit) : sum;
            g.lse[head * g.lse_sh + seq.pq + at] =
                at < seq.nq && z != 0.0f ? m[qb] + log2f(z) : INFINITY;
        }
        if (at >= seq.eq) continue;
        const float f = at < seq.nq && sum != 0.0f ? unit / sum : 0.0f;
        const int64_t to = sid * g.out.sb + (seq.q0 + at) * g.out.sr + head * g.out.sh;
        const bool vec = g.out.sd == 1 && g.dim % 4 == 0;
#pragma unroll
        for (int fb = 0; fb < DB; ++fb) {
            // a row that sees no key, or is no query: zeros
            f32x16 x = o[fb][qb];
            if (f == 0.0f) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 0.0f;
            }
            if (g.dtype == SLK_F32) attn_store<F32>(g.out, to, fb, lane, g.dim, vec, x, f);
            else attn_store<BF16>(g.out, to, fb, lane, g.dim, vec, x, f);
        }
    }
}

// Joins the parts of split keys: one workgroup of 64 threads a query and head.
__global__ __launch_bounds__(kWave) void attn_join_kernel(const AttnArgs g, int dp) {
    const int64_t row = blockIdx.x;
    const int head = blockIdx.y, lane = threadIdx.x;
    // padded row -> sequence
    int sid = 0, at = 0;
    AttnSeq seq;
    if (g.plan.seqs == nullptr) {
        sid = static_cast<int>(row / g.plan.pad_t);
        at = static_cast<int>(row - sid * g.plan.pad_t);
        seq = attn_seq(g.plan, sid);
    } else {
        int lo = 0, hi = static_cast<int>(g.plan.batch);
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (g.plan.seqs[mid].pq <= row) lo = mid;
            else hi = mid;
        }
        sid = lo;
        seq = g.plan.seqs[sid];
        at = static_cast<int>(row) - seq.pq;
    }
    if (at >= seq.nq) {
        // padding's log-sum, and rows that are written but are no queries
        if (g.lse != nullptr && lane == 0) g.lse[head * g.lse_sh + row] = INFINITY;
        return;
    }
    float top = -INFINITY;
    for (int s = 0; s < g.splits; ++s) {
        const int64_t r = (static_cast<int64_t>(s) * g.heads + head) * g.part_rows + row;
        top = fmaxf(top, g.part_ml[2 * r]);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, x[2] = {0.0f, 0.0f};
    for (int s = 0; s < g.splits; ++s) {
        const int64_t r = (static_cast<int64_t>(s) * g.heads + head) * g.part_rows + row;
        const float part = g.part_ml[2 * r + 1];
        if (part == 0.0f) continue;  // saw no key (its maximum is -inf)
        const float a = attn_exp2(g.part_ml[2 * r] - ref);
        sum = __builtin_fmaf(part, a, sum);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int f = lane + 64 * j;
            if (f < dp) x[j] = __builtin_fmaf(g.part[r * dp + f], a, x[j]);
        }
    }
    if (g.lse != nullptr && lane == 0)
        g.lse[head * g.lse_sh + row] = sum != 0.0f ? top + log2f(sum) : INFINITY;
    const int64_t to = sid * g.out.sb + (seq.q0 + at) * g.out.sr + head * g.out.sh;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int f = lane + 64 * j;
        if (f >= g.dim) continue;
        const float y = sum != 0.0f ? x[j] / sum : 0.0f;
        if (g.dtype == SLK_F32) F32::store(g.out.p, to + f * g.out.sd, y);
        else BF16::store(g.out.p, to + f * g.out.sd, y);
    }
}

template <bool SPLIT, int DB, int QB>
int launch(const AttnArgs& g, int64_t entries, hipStream_t st) {
    const int64_t groups = entries * g.splits * g.heads;
    if (groups > max_groups(kAttnThreads))
        return fail(SLK_EINVAL, "attention_forward: too many query tiles");
    const dim3 grid(static_cast<unsigned>(groups)), wg(kAttnThreads);
    if (g.bias.table != nullptr) {
        const size_t lds = (2 * g.bias.max_distance + 1) * sizeof(float);
        hipLaunchKernelGGL((attn_forward_kernel<SPLIT, DB, QB, true>), grid, wg, lds, st, g);
    } else {
        hipLaunchKernelGGL((attn_forward_kernel<SPLIT, DB, QB, false>), grid, wg, 0, st, g);
    }
    int rc = check_launch("attention_forward");
    if (rc != SLK_OK || g.splits == 1) return rc;
    return attn_launch_join(g, DB, st);
}

}  // namespace

int attn_launch_join(const AttnArgs& g, int db, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(g.part_rows), g.heads);
    hipLaunchKernelGGL(attn_join_kernel, grid, dim3(kWave), 0, st, g, 32 * db);
    return check_launch("attention_forward: join");
}

int attn_launch_forward(const AttnArgs& g, bool split, int db, int64_t entries, hipStream_t st) {
    if (split) {
        return db == 1   ? launch<true, 1, 1>(g, entries, st)
               : db == 2 ? launch<true, 2, 1>(g, entries, st)
                         : launch<true, 4, 1>(g, entries, st);
    }
    return db == 1   ? launch<false, 1, 1>(g, entries, st)
           : db == 2 ? launch<false, 2, 1>(g, entries, st)
                     : launch<false, 4, 1>(g, entries, st);
}

}  // namespace slk
