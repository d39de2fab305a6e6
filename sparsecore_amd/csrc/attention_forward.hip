// slk_attention_forward's kernel.
#include "attention.hpp"
#include "elem.hpp"

namespace slk {

namespace {

// Largest growth (in log 2) of a row's maximum that is left in its exponentials
// before the row is rescaled, and where packed weights start: below 2^15 in all.
constexpr float kGrowth = 8.0f;
constexpr int kWeightUnit = 7;

// A workgroup takes 128 queries of one head, a wave 32 of them; keys and values
// come through LDS, 64 at a time, two buffers, one barrier a tile. The scores are
// computed as K·Q^T, so that a lane holds half of a query's 64 (the others are 32
// lanes away): the softmax's maximum and sum are the lane's own, and its weights
// are the operand of O^T = V^T·P^T as they are. The row's maximum is only raised
// when a new one is more than 2^8 times above. O has a unit of its own, 2^ev, as a tile's
// values are in units of their largest: of the largest weight times value so far, row by
// row, so that neither a tile that a row does not see nor one of large values that it
// hardly looks at takes bits off its weights. One sequence of 16384, 32 heads over 8
// of 128, bfloat16, causal: 2.2 ms, 1.0 PFLOP/s (a large library product of bfloat16
// reaches 1.24), bound by the matrix cores and the exponentials between them.
template <bool SPLIT, int DB, bool BIAS>
__global__ __launch_bounds__(kAttnThreads, DB * (SPLIT ? 2 : 1) <= 4 ? 2 : 1) void
attn_forward_kernel(const AttnArgs g) {
    using T = AttnTile<DB>;
    constexpr int kBytes = (SPLIT ? 2 : 1) * T::kPlane, KS = 2 * DB;
    __shared__ __align__(16) unsigned char ring0[2 * kBytes];
    __shared__ __align__(16) unsigned char ring1[2 * kBytes];
    extern __shared__ float bias_row[];

    const int t = threadIdx.x, lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t rep = g.heads / g.kv_heads;
    const uint32_t kvh = blockIdx.x % g.kv_heads, u0 = blockIdx.x / g.kv_heads;
    const uint32_t hg = u0 % rep, u1 = u0 / rep;
    const int split = static_cast<int>(u1 % g.splits);
    const int head = static_cast<int>(kvh * rep + hg);
    int sid, tile;
    if (!attn_entry(g.plan, u1 / g.splits, g.tiles, false, sid, tile)) return;
    const AttnSeq seq = attn_seq(g.plan, sid);
    const int rows0 = tile * 128, shift = seq.nk - seq.nq;
    const int wave0 = rows0 + 32 * wv;
    const int q = wave0 + (lane & 31);

    // keys that the workgroup's queries see, and this part's share of their tiles
    const int last_q = min(rows0 + 128, seq.nq) - 1;
    const int seen = last_q < rows0 ? 0 : g.causal ? min(seq.nk, last_q + shift + 1) : seq.nk;
    const int n_tiles = seen <= 0 ? 0 : (seen + kAttnRows - 1) / kAttnRows;
    const int per = (n_tiles + g.splits - 1) / g.splits;
    const int t0 = min(split * per, n_tiles), t1 = min(t0 + per, n_tiles);

    float m = -INFINITY, l = 0.0f;
    f32x16 o[DB];
#pragma unroll
    for (int fb = 0; fb < DB; ++fb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[fb][r] = 0.0f;
    int ev = kUnset;

    if (t0 < t1) {
        const char* const kp = g.k.p + kvh * g.k.sh + static_cast<int64_t>(seq.pk / 64) * kBytes;
        const char* const vp = g.v.p + kvh * g.v.sh + static_cast<int64_t>(seq.pk / 64) * kBytes;
        auto issue = [&](AttnLds* to, int kt) __attribute__((always_inline)) {
            attn_stage<kBytes>(kp + static_cast<int64_t>(kt) * kBytes, to, wv, lane);
            attn_stage<kBytes>(vp + static_cast<int64_t>(kt) * kBytes, to + kBytes, wv, lane);
        };
        issue((AttnLds*)ring0, t0);
        const AttnReads<SPLIT, DB> rd(lane);

        const int q_row = seq.pq + min(wave0, (seq.nq + 63) / 64 * 64 - 32);
        const int even_qe = attn_exp(g.q, head, q_row);
        AttnPair<SPLIT> qf[KS];
        {
            const unsigned char* at = reinterpret_cast<const unsigned char*>(
                g.q.p + head * g.q.sh + static_cast<int64_t>(q_row / 64) * kBytes);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[ks] = rd.along(at, (q_row >> 5) & 1, ks);
        }
        const int tiles0 = seq.pk / 64;
        if constexpr (BIAS) attn_bias_row(g.bias, head, bias_row);
        const int md = BIAS ? g.bias.max_distance : 0;

        // ROWS: exponents row by row, as uneven tiles have them
        auto compute = [&](auto rows, const unsigned char* buf, int kt)
            __attribute__((always_inline)) {
            constexpr bool ROWS = decltype(rows)::value;
            const int key0 = kt * kAttnRows;
            // the wave's last query sees no key of this tile
            if (g.causal && key0 > wave0 + 31 + shift) return;
            const bool masked = key0 + 63 >= seq.nk || (g.causal && key0 + 63 > wave0 + shift);
            f32x16 s[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.0f;
            attn_pipeline<SPLIT, 2 * KS, kAttnAhead<SPLIT>>(
                [&](auto i) __attribute__((always_inline)) {
                    return rd.along(buf, i.value % 2, i.value / 2);
                },
                [&](auto i, const AttnPair<SPLIT>& k) __attribute__((always_inline)) {
                    s[i.value % 2] = attn_dot<SPLIT>(k, qf[i.value / 2], s[i.value % 2]);
                });
            const int64_t et = kvh * g.k.exps_sh + tiles0 + kt;
            const int qe = ROWS ? *g.q.row(head, q_row + (lane & 31)) : even_qe;
            const int ve = attn_scalar(g.v.exps + et), ke = attn_scalar(g.k.exps + et);
            float c = 1.0f;
            if constexpr (ROWS) {
                const int8_t* const at = g.k.row(kvh, seq.pk + key0 + 4 * (lane >> 5));
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    const uint32_t four = attn_four_rows(at + 8 * (r / 4));
                    s[r / 16][r % 16] =
                        ldexpf(s[r / 16][r % 16] * g.scale2,
                               qe + attn_one_of(four, r % 4) - 2 * kAttnUnit);
                }
            } else {
                // not beyond float32: a row of zeros has scores of 0
                c = ldexpf(g.scale2, min(qe + (ke >> 2) - 2 * kAttnUnit, 126));
            }
            // the last key that this query sees, from the tile's first
            const int lim = (g.causal ? min(seq.nk - 1, q + shift) : seq.nk - 1) - key0;
            if constexpr (BIAS) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const int lo = wave0 + shift - key0 - 32 * kb - 31, hi = lo + 62;
                    if (lo >= md || hi <= -md) {
                        const float b = bias_row[kAttnFar + (lo >= md ? 2 * md : 0)];
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(s[kb][r], c, b);
                    } else {
                        // key 27 of the block's lane rows on, then back to the first
                        const float* const at = bias_row + md + kAttnFar + q + shift - key0 -
                                                32 * kb - 4 * (lane >> 5) - 27;
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[kb][r] =
                                __builtin_fmaf(s[kb][r], c, at[27 - 8 * (r >> 2) - (r & 3)]);
                    }
                }
                c = 1.0f;
            }
            if (masked) {  // scaled first: the factor may be 0
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[kb][r] = 32 * kb + attn_row(r, lane) <= lim ? s[kb][r] * c : -INFINITY;
                c = 1.0f;
            }
            float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(fmaxf(s[0][r], s[1][r]), top);
            top = fmaxf(top, __shfl_xor(top, 32)) * c;
            // The largest weight times value, from the row's maximum: as a tile's exponent or
            // row by row. Differences first: a bias of the lowest value would swallow what is
            // added to it.
            const int8_t* const v_rows = g.v.row(kvh, seq.pk + key0 + 4 * (lane >> 5));
            const float up = fmaxf(m, top);
            float most = top - up + static_cast<float>(ve >> 2), over;
            if constexpr (ROWS) {
                most = -INFINITY;
                const float from = up == -INFINITY ? 0.0f : up;
#pragma unroll
                for (int r = 0; r < 32; ++r)
                    most = fmaxf(most, s[r / 16][r % 16] - from +
                                           static_cast<float>(attn_one_of(
                                               attn_four_rows(v_rows + 8 * (r / 4)), r % 4)));
                most = fmaxf(most, __shfl_xor(most, 32));
                over = up - m + fmaxf(most - static_cast<float>(ev), 0.0f);
            } else {
                over = top - m + static_cast<float>(max((ve >> 2) - ev, 0));
            }
            if (__builtin_amdgcn_ballot_w64(over > kGrowth) != 0) {
                if (up > -INFINITY) {
                    // O shrinks with the weights: by whole powers of two its unit does. The
                    // fraction of a power of two is the same factor for the sum and for O.
                    const float grow = fminf(up - m, 1000.0f);
                    const int whole = static_cast<int>(grow);
                    const int mine = static_cast<int>(ceilf(fmaxf(most, -1000.0f)));
                    const int to = max(m > -INFINITY ? ev - whole : kUnset,
                                       top > -INFINITY ? mine : kUnset);
                    const float part = attn_exp2(static_cast<float>(whole) - grow);
                    l *= m > -INFINITY ? ldexpf(part, -whole) : 0.0f;
                    const float a = m > -INFINITY ? ldexpf(part, ev - to - whole) : 0.0f;
#pragma unroll
                    for (int fb = 0; fb < DB; ++fb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[fb][r] *= a;
                    m = up;
                    ev = to;
                }
            }
            // weights times 2^(unit + d): values of a smaller exponent weigh less
            const int d = ROWS ? 0 : max((ve >> 2) - ev, -60);
            const float ref = m == -INFINITY ? 0.0f : m, unit = static_cast<float>(kWeightUnit + d);
            const float start = unit - ref;
            float sum = 0.0f;
            AttnPair<SPLIT> w[2][2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                float p[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if constexpr (ROWS) {
                        const float x = s[kb][r] - ref;
                        sum += attn_exp2(x);
                        const uint32_t four = attn_four_rows(v_rows + 32 * kb + 8 * (r / 4));
                        p[r] = attn_exp2(x + static_cast<float>(attn_one_of(four, r % 4) - ev +
                                                                kWeightUnit));
                        continue;
                    }
                    // a bias may be large enough to swallow the unit: it comes second
                    if constexpr (BIAS) p[r] = attn_exp2(__builtin_fmaf(s[kb][r], c, -ref) + unit);
                    else p[r] = attn_exp2(__builtin_fmaf(s[kb][r], c, start));
                    sum += p[r];
                }
                w[kb][0] = attn_operand<SPLIT>(p);
                w[kb][1] = attn_operand<SPLIT>(p + 8);
            }
            l = __builtin_fmaf(sum, attn_pow2(ROWS ? kWeightUnit : -d), l);
            if (__builtin_expect((ve | ke) & 1, 0)) {  // rows that are not finite
                const uint64_t bad = attn_scalar(g.v.bad + et) | attn_scalar(g.k.bad + et);
                const uint64_t sees = lim >= 63 ? ~uint64_t{0}
                                      : lim >= 0 ? (uint64_t{2} << lim) - 1
                                                 : 0;
                if (bad & sees) l = __builtin_nanf("");
            }
            attn_accumulate<SPLIT, DB, 2>(rd, buf + kBytes, 0, w, o);
        };
        auto stage = [&](auto rows, const unsigned char* cur, unsigned char* next, int kt)
            __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(wait_vm(0));
            asm volatile("s_barrier" ::: "memory");
            if (kt + 1 < t1) issue((AttnLds*)next, kt + 1);
            if (wave0 < seq.nq) compute(rows, cur, kt);
        };
        auto all = [&](auto rows) __attribute__((always_inline)) {
            int kt = t0;
            for (; kt + 2 <= t1; kt += 2) {
                stage(rows, ring0, ring1, kt);
                stage(rows, ring1, ring0, kt + 1);
            }
            if (kt < t1) stage(rows, ring0, ring1, kt);
        };
        // of all the tiles that the workgroup meets
        const int64_t q0 = (seq.pq + rows0) / kAttnRows, q1 = q0 + (min(seq.nq - rows0, 128) + 63) / 64;
        if (attn_uneven(attn_flags(g.q, head, q0, q1, lane) |
                        attn_flags(g.k, kvh, tiles0 + t0, tiles0 + t1, lane) |
                        attn_flags(g.v, kvh, tiles0 + t0, tiles0 + t1, lane) |
                        attn_more_flags(g.k, kvh, tiles0 + t0, tiles0 + t1, lane) |
                        attn_more_flags(g.v, kvh, tiles0 + t0, tiles0 + t1, lane)))
            all(std::true_type{});
        else all(std::false_type{});
    }

    float sum = l + __shfl_xor(l, 32);
    if (t0 < t1 && q < seq.nq) {
        const int64_t et = head * g.q.exps_sh + ((seq.pq + q) >> 6);
        if ((g.q.exps[et] & 1) && ((g.q.bad[et] >> (q & 63)) & 1) && sum != 0.0f)
            sum = __builtin_nanf("");
    }
    if (g.splits > 1 && q < seq.nq) {
        const int64_t row =
            (static_cast<int64_t>(split) * g.heads + head) * g.part_rows + seq.pq + q;
        if (lane < 32) {
            g.part_ml[2 * row] = m;
            g.part_ml[2 * row + 1] = sum * attn_pow2(-kWeightUnit);
        }
        const float f = attn_pow2(ev - kAttnUnit - kWeightUnit);
#pragma unroll
        for (int fb = 0; fb < DB; ++fb)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                f32x4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = o[fb][4 * r4 + j] * f;
                *reinterpret_cast<f32x4*>(g.part + row * T::DP + 32 * fb + 8 * r4 +
                                          4 * (lane >> 5)) = x;
            }
        return;
    }
    if (split != 0) return;  // the first part writes what no query stands behind
    if (g.lse != nullptr && lane < 32 && g.splits == 1 && q < (seq.nq + 63) / 64 * 64) {
        const int64_t at = head * g.lse_sh + seq.pq + q;
        const bool any = q < seq.nq && sum != 0.0f;
        const float s = sum * attn_pow2(-kWeightUnit);
        if constexpr (BIAS) {
            g.lse[at] = any ? (s == s ? m : s) : INFINITY;
            g.inv[at] = any ? 1.0f / s : 0.0f;
        } else {
            g.lse[at] = any ? m + log2f(s) : INFINITY;
        }
    }
    if (q >= seq.eq) return;
    const bool zero = q >= seq.nq || sum == 0.0f;  // no query, or one that sees no key
    const float f = zero ? 0.0f : attn_pow2(ev - kAttnUnit) / sum;
    const int64_t to = sid * g.out.sb + (seq.q0 + q) * g.out.sr + head * g.out.sh;
    const bool vec = g.out.sd == 1 && g.vec_out;
#pragma unroll
    for (int fb = 0; fb < DB; ++fb) {
        f32x16 x = o[fb];
        if (zero) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = 0.0f;
        }
        if (g.dtype == SLK_F32) attn_store<F32>(g.out, to, fb, lane, g.dim, vec, x, f);
        else attn_store<BF16>(g.out, to, fb, lane, g.dim, vec, x, f);
        if (g.o_rest != nullptr && q < seq.nq) {
            const int64_t row = head * g.lse_sh + seq.pq + q;
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                float rest[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y = x[4 * r4 + j] * f;
                    rest[j] = y - bf16_to_f32(f32_to_bf16(y));
                }
                BF16::store4(g.o_rest,
                             attn_rest_at(row, 32 * fb + 8 * r4 + 4 * (lane >> 5), T::DP), rest);
            }
        }
    }
}

// Joins the parts of split keys: a wave a query and head. Its lanes read the parts'
// maxima and sums side by side; then each sixteen lanes add up every fourth part,
// four features a lane.
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(const AttnArgs g, int dp) {
    const int lane = threadIdx.x & 63, head = blockIdx.y;
    const int64_t rows = g.plan.seqs != nullptr ? g.part_rows : g.plan.batch * g.plan.t;
    const int64_t e = static_cast<int64_t>(blockIdx.x) * (kAttnThreads / 64) + threadIdx.x / 64;
    if (e >= rows) return;
    int sid, at;
    AttnSeq seq;
    int64_t row;
    if (g.plan.seqs == nullptr) {
        sid = static_cast<int>(e / g.plan.t);
        at = static_cast<int>(e - sid * g.plan.t);
        seq = attn_seq(g.plan, sid);
        row = seq.pq + at;
    } else {
        row = e;
        const AttnRow r = attn_row_of(g.plan, false, row);
        if (!r.any || r.row >= r.seq.nq) return;
        sid = r.sid;
        at = r.row;
        seq = r.seq;
    }
    const int64_t step = static_cast<int64_t>(g.heads) * g.part_rows;
    const int64_t r0 = head * g.part_rows + row;
    constexpr int kMost = kAttnMaxSplits / 64;
    float top = -INFINITY, mine[kMost], sums[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int s = lane + 64 * i;
        mine[i] = -INFINITY;
        sums[i] = 0.0f;
        if (s < g.splits) {
            const float2 x = *reinterpret_cast<const float2*>(g.part_ml + 2 * (r0 + s * step));
            mine[i] = x.x;
            sums[i] = x.y;
        }
        top = fmaxf(top, mine[i]);
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        // a part that saw no key has sum 0 (and maximum -inf)
        mine[i] = sums[i] == 0.0f ? 0.0f : attn_exp2(mine[i] - top);
        sum += sums[i] == 0.0f ? 0.0f : sums[i] * mine[i];
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
    const float inv = 1.0f / sum;
    const int64_t to = sid * g.out.sb + (seq.q0 + at) * g.out.sr + head * g.out.sh;
    for (int f0 = 0; f0 < dp; f0 += 64) {
        const int f = f0 + 4 * (lane & 15);
        const float* p = g.part + r0 * dp + (f < dp ? f : 0);
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int s0 = 0; s0 < g.splits; s0 += 4) {
            const int s = s0 + (lane >> 4);
            const float w = __shfl(s0 < 64 ? mine[0] : mine[1], s & 63);
            const f32x4 y =
                *reinterpret_cast<const f32x4*>(p + min(s, g.splits - 1) * step * dp);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[j] = __builtin_fmaf(y[j], s < g.splits ? w : 0.0f, x[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] += __shfl_xor(x[j], 16);
            x[j] += __shfl_xor(x[j], 32);
        }
        if (lane >= 16 || f >= dp) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (f + j >= g.dim) break;
            const float y = sum != 0.0f ? x[j] * inv : 0.0f;
            if (g.dtype == SLK_F32) F32::store(g.out.p, to + (f + j) * g.out.sd, y);
            else BF16::store(g.out.p, to + (f + j) * g.out.sd, y);
        }
    }
}
static_assert(kAttnMaxSplits == 128, "two parts a lane");

template <bool SPLIT, int DB>
int launch(const AttnArgs& g, int64_t entries, hipStream_t st) {
    const int64_t groups = entries * g.splits * g.heads;
    if (groups > max_groups(kAttnThreads))
        return fail(SLK_EINVAL, "attention_forward: too many query tiles");
    const dim3 grid(static_cast<unsigned>(groups)), wg(kAttnThreads);
    if (g.bias.table != nullptr) {
        const size_t lds = attn_bias_floats(g.bias.max_distance) * sizeof(float);
        hipLaunchKernelGGL((attn_forward_kernel<SPLIT, DB, true>), grid, wg, lds, st, g);
    } else {
        hipLaunchKernelGGL((attn_forward_kernel<SPLIT, DB, false>), grid, wg, 0, st, g);
    }
    int rc = check_launch("attention_forward");
    if (rc != SLK_OK || g.splits == 1) return rc;
    return attn_launch_join(g, DB, st);
}

}  // namespace

int attn_launch_join(const AttnArgs& g, int db, hipStream_t st) {
    const int64_t rows = g.plan.seqs != nullptr ? g.part_rows : g.plan.batch * g.plan.t;
    const dim3 grid(static_cast<unsigned>(ceil_div(rows, kAttnThreads / 64)), g.heads);
    hipLaunchKernelGGL(attn_join_kernel, grid, dim3(kAttnThreads), 0, st, g, 32 * db);
    return check_launch("attention_forward: join");
}

int attn_launch_forward(const AttnArgs& g, bool split, int db, int64_t entries, hipStream_t st) {
    if (split) {
        return db == 1   ? launch<true, 1>(g, entries, st)
               : db == 2 ? launch<true, 2>(g, entries, st)
                         : launch<true, 4>(g, entries, st);
    }
    return db == 1   ? launch<false, 1>(g, entries, st)
           : db == 2 ? launch<false, 2>(g, entries, st)
                     : launch<false, 4>(g, entries, st);
}

}  // namespace slk
