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

// One workgroup. Offsets that fall, or pass the arrays' end, are taken as the
// nearest ones that do not: no row is written twice or outside.
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
    const bool one_each = total <= kPlanThreads;  // a thread keeps its sequence
    const AttnSeq own = one_each && t < total ? a.seqs[t] : AttnSeq{};
    for (int side = 0; side < 2; ++side) {
        int2* list = side ? a.k_list : a.q_list;
        if (list == nullptr) continue;
        auto each = [&](auto&& f) {
            for (int s = t; s < total; s += kPlanThreads) {
                const AttnSeq x = one_each ? own : a.seqs[s];
                const int shift = x.nk - x.nq;
                const int tiles = ((side ? x.ek : x.eq) + kTileRows - 1) / kTileRows;
                for (int i = 0; i < tiles; ++i) {
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

struct RowOf {
    int sid, row;  // row of the sequence; at or past its last live row: none
    AttnSeq seq;
    bool any;
};

// Sequence and row of a padded row of queries or keys.
__device__ __forceinline__ RowOf row_of(const AttnPlan& p, bool keys, int64_t padded) {
    RowOf r;
    if (p.seqs == nullptr) {
        const int64_t pad = keys ? p.pad_s : p.pad_t;
        r.sid = static_cast<int>(padded / pad);
        r.any = r.sid < p.batch;
        r.seq = attn_seq(p, r.sid);
        r.row = static_cast<int>(padded - r.sid * pad);
        return r;
    }
    r.any = padded < p.count[keys ? 3 : 1];
    int lo = 0, hi = static_cast<int>(p.batch);
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((keys ? p.seqs[mid].pk : p.seqs[mid].pq) <= padded) lo = mid;
        else hi = mid;
    }
    r.sid = lo;
    r.seq = p.seqs[lo];
    r.row = static_cast<int>(padded - (keys ? r.seq.pk : r.seq.pq));
    return r;
}

// Packs a tile of 64 rows of one head: blockIdx.x the tile, blockIdx.y the head of
// an operand; one more y for the rows of biases, a head each. Lanes run along
// whichever of rows and features is consecutive in memory. Of dO (with delta
// given) also delta, from the same tile and O. What bounds it is memory.
template <bool SPLIT, int DB, class IO>
__global__ __launch_bounds__(kAttnThreads) void attn_pack_kernel(const AttnPack a) {
    constexpr int DP = 32 * DB;
    __shared__ float x[kAttnRows][DP + 1];
    __shared__ int32_t top;
    __shared__ uint32_t odd[2];  // rows with a value that is not finite
    const int t = threadIdx.x;
    int which = 0, head = blockIdx.y;
    while (which < a.n && head >= a.op[which].heads) head -= a.op[which++].heads;
    if (which == a.n) {
        const int width = 2 * a.bias.max_distance + 1;
        for (int h = blockIdx.x; h < a.heads; h += gridDim.x)
            for (int i = t; i < width; i += kAttnThreads)
                a.bias.rows[static_cast<int64_t>(h) * width + i] =
                    attn_bias_of(a.bias, a.heads, h, i - a.bias.max_distance);
        return;
    }
    const AttnPackOp& op = a.op[which];
    const int64_t padded = static_cast<int64_t>(blockIdx.x) * kAttnRows;
    if (padded >= op.rows) return;
    const RowOf ro = row_of(a.plan, op.keys, padded);
    if (!ro.any) return;
    const int n = op.keys ? ro.seq.nk : ro.seq.nq, first = op.keys ? ro.seq.k0 : ro.seq.q0;
    const int live = min(max(n - ro.row, 0), kAttnRows);
    const int64_t row = first + ro.row;
    if (t == 0) top = odd[0] = odd[1] = 0;
    __syncthreads();
    const int64_t at = ro.sid * op.src.sb + row * op.src.sr + head * op.src.sh;
    uint32_t m = 0;  // the largest finite magnitude
    auto put = [&](int r, int f, float v) {
        const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
        if (b < 0x7f800000u) {
            m = max(m, b);
        } else {
            v = 0.0f;
            atomicOr(&odd[r >> 5], 1u << (r & 31));
        }
        x[r][f] = v;
    };
    if (op.vec == kVecFeatures) {
        for (int i = t; i < kAttnRows * DP / 4; i += kAttnThreads) {
            const int r = i / (DP / 4), f = 4 * (i % (DP / 4));
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (r < live && f < a.dim) IO::load4(op.src.p, at + r * op.src.sr + f, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) put(r, f + j, v[j]);
        }
    } else if (op.vec == kVecRows) {
        for (int i = t; i < kAttnRows * DP / 4; i += kAttnThreads) {
            const int r = 4 * (i % (kAttnRows / 4)), f = i / (kAttnRows / 4);
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int64_t from = at + r + f * op.src.sd;
            if (f < a.dim) {
                // four rows at once where they are aligned and all live
                if (r + 4 <= live && ((row + r) & 3) == 0) {
                    IO::load4(op.src.p, from, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (r + j < live) v[j] = IO::load(op.src.p, from + j);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) put(r + j, f, v[j]);
        }
    } else {
        const bool rows_first = op.src.sr == 1 && op.src.sd != 1;
        for (int i = t; i < kAttnRows * DP; i += kAttnThreads) {
            const int r = rows_first ? i % kAttnRows : i / DP;
            const int f = rows_first ? i / kAttnRows : i % DP;
            float v = 0.0f;
            if (r < live && f < a.dim) v = IO::load(op.src.p, at + r * op.src.sr + f * op.src.sd);
            put(r, f, v);
        }
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(m, s)));
    __syncthreads();
    if ((t & 63) == 0) atomicMax(&top, static_cast<int>(m));
    __syncthreads();
    const int e = max(static_cast<int>(static_cast<uint32_t>(top) >> 23) - 127, -100);
    const uint64_t bad = static_cast<uint64_t>(odd[1]) << 32 | odd[0];
    if (t == 0) {
        op.exps[head * op.exps_sh + padded / kAttnRows] = 2 * e + (bad != 0 ? 1 : 0);
        op.bad[head * op.exps_sh + padded / kAttnRows] = bad;
    }

    // rows in pieces of eight features, permuted as they will lie in LDS
    using T = AttnTile<DB>;
    const float factor = ldexpf(1.0f, kAttnUnit - e);
    char* const to = op.dst + head * op.dst_sh +
                     static_cast<int64_t>(blockIdx.x) * ((SPLIT ? 2 : 1) * T::kPlane);
    for (int i = t; i < kAttnRows * T::kPieces; i += kAttnThreads) {
        const int r = i / T::kPieces, c = (i % T::kPieces) ^ T::swz(r);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[r][8 * c + j] * factor;
        const AttnPair<SPLIT> f = attn_operand<SPLIT>(v);
        *reinterpret_cast<f16x8*>(to + 16 * i) = f.f[0];
        if constexpr (SPLIT) *reinterpret_cast<f16x8*>(to + T::kPlane + 16 * i) = f.f[1];
    }

    if (a.delta == nullptr) return;
    __syncthreads();
    if (t == 0) top = 0;
    __syncthreads();
    // delta: lanes over rows where O's rows are consecutive, else four lanes a row
    const bool rows_first = a.o.sr == 1 && a.o.sd != 1;
    const int r = rows_first ? t % 64 : t / 4, part = rows_first ? t / 64 : t % 4;
    float d = 0.0f;
    const int64_t from = ro.sid * a.o.sb + (row + r) * a.o.sr + head * a.o.sh;
    if (r < live) {
        if (a.o_vec && !rows_first) {
            for (int f = 4 * part; f < a.dim; f += 16) {
                float v[4];
                IO::load4(a.o.p, from + f, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) d = __builtin_fmaf(x[r][f + j], v[j], d);
            }
        } else {
            for (int f = part; f < a.dim; f += 4)
                d = __builtin_fmaf(x[r][f], IO::load(a.o.p, from + f * a.o.sd), d);
        }
    }
    __syncthreads();
    float* const sums = &x[0][0];
    sums[4 * r + part] = d;
    __syncthreads();
    if (t < kAttnRows) {
        const float y = (sums[4 * t] + sums[4 * t + 1]) + (sums[4 * t + 2] + sums[4 * t + 3]);
        const int64_t at_row = head * a.delta_sh + padded + t;
        a.delta[at_row] = y;
        a.lse_out[at_row] = (bad >> t) & 1 ? __builtin_nanf("") : a.lse[at_row];
        uint32_t b = __float_as_uint(y) & 0x7fffffffu;
        b = b < 0x7f800000u ? b : 0;
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) b = max(b, static_cast<uint32_t>(__shfl_xor(b, s)));
        if (t == 0)
            a.dexps[head * op.exps_sh + padded / kAttnRows] =
                max(static_cast<int>(b >> 23) - 127, -100);
    }
}

template <bool SPLIT, class IO>
int pack(const AttnPack& a, int db, dim3 grid, hipStream_t st) {
    const dim3 wg(kAttnThreads);
    if (db == 1) hipLaunchKernelGGL((attn_pack_kernel<SPLIT, 1, IO>), grid, wg, 0, st, a);
    else if (db == 2) hipLaunchKernelGGL((attn_pack_kernel<SPLIT, 2, IO>), grid, wg, 0, st, a);
    else hipLaunchKernelGGL((attn_pack_kernel<SPLIT, 4, IO>), grid, wg, 0, st, a);
    return check_launch("attention: pack");
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
