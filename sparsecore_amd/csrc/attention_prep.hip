// What comes before the attention kernels: the sequences' table and tile order,
// operands in 16-bit parts, and the backward's row sums of dO∘O.
#include "attention.hpp"
#include "attention_prep.hpp"
#include "elem.hpp"

namespace slk {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kBins = 1024;  // classes of work in the tile order

// Inclusive scan over the workgroup, by sum or maximum.
template <bool MAX>
__device__ int64_t scan(int64_t x, int64_t* lds) {
    const int t = threadIdx.x;
    lds[t] = x;
    __syncthreads();
    for (int o = 1; o < kPlanThreads; o <<= 1) {
        const int64_t y = t >= o ? lds[t - o] : (MAX ? INT64_MIN : 0);
        __syncthreads();
        x = MAX ? (x > y ? x : y) : x + y;
        lds[t] = x;
        __syncthreads();
    }
    return x;
}

// One workgroup. Offsets that fall, or pass the arrays' end, are taken as the
// nearest ones that do not: no row is written twice or outside.
__global__ __launch_bounds__(kPlanThreads) void attn_plan_kernel(const AttnPlanArgs a) {
    __shared__ int64_t lds[kPlanThreads];
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
            // starts: running maximum of the offsets so far, ends: with the next one
            const int64_t oq = in ? clamp(a.q_offsets[s], a.rows_q) : 0;
            const int64_t ok = in ? clamp(a.k_offsets[s], a.rows_k) : 0;
            int64_t bq = scan<true>(oq, lds);
            __syncthreads();
            int64_t bk = scan<true>(ok, lds);
            __syncthreads();
            bq = bq > endq ? bq : endq;
            bk = bk > endk ? bk : endk;
            const int64_t nq = in ? clamp(a.q_offsets[s + 1], a.rows_q) : 0;
            const int64_t nk = in ? clamp(a.k_offsets[s + 1], a.rows_k) : 0;
            x.q0 = static_cast<int32_t>(bq);
            x.k0 = static_cast<int32_t>(bk);
            x.nq = x.eq = static_cast<int32_t>(nq > bq ? nq - bq : 0);
            x.nk = x.ek = static_cast<int32_t>(nk > bk ? nk - bk : 0);
            int64_t lq = scan<true>(in ? bq + x.nq : 0, lds);
            lds[t] = lq;
            __syncthreads();
            lq = lds[kPlanThreads - 1];
            __syncthreads();
            int64_t lk = scan<true>(in ? bk + x.nk : 0, lds);
            lds[t] = lk;
            __syncthreads();
            lk = lds[kPlanThreads - 1];
            __syncthreads();
            endq = lq > endq ? lq : endq;
            endk = lk > endk ? lk : endk;
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
        const int64_t iq = scan<false>(wq, lds);
        const int64_t totq = lds[kPlanThreads - 1];
        __syncthreads();
        const int64_t ik = scan<false>(wk, lds);
        const int64_t totk = lds[kPlanThreads - 1];
        __syncthreads();
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
    const int64_t total = a.n + (packed ? 2 : 0);
    for (int side = 0; side < 2; ++side) {
        int2* list = side ? a.k_list : a.q_list;
        if (list == nullptr) continue;
        const int rows = side ? a.tile_k : a.tile_q;
        auto each = [&](auto&& f) {
            for (int64_t s = t; s < total; s += kPlanThreads) {
                const AttnSeq x = a.seqs[s];
                const int shift = x.nk - x.nq;
                const int tiles = static_cast<int>(ceil_div(side ? x.ek : x.eq, rows));
                for (int i = 0; i < tiles; ++i) {
                    int64_t w;
                    if (side) {
                        w = x.nk <= i * rows ? 0
                            : a.causal       ? x.nq - max(0, i * rows - shift)
                                             : x.nq;
                    } else {
                        w = x.nq <= i * rows ? 0
                            : a.causal       ? min(x.nk, min((i + 1) * rows, x.nq) + shift)
                                             : x.nk;
                    }
                    w = ceil_div(w < 0 ? 0 : w, kAttnRows) >> a.work_shift;
                    f(static_cast<int>(kBins - 1 - (w < kBins ? w : kBins - 1)),
                      static_cast<int>(s), i);
                }
            }
        };
        for (int i = t; i < kBins; i += kPlanThreads) bin[i] = 0;
        __syncthreads();
        each([&](int b, int, int) { atomicAdd(&bin[b], 1); });
        __syncthreads();
        const int64_t mine = bin[t];
        const int64_t upto = scan<false>(mine, lds);
        const int64_t all = lds[kPlanThreads - 1];
        bin[t] = static_cast<int32_t>(upto - mine);
        __syncthreads();
        // the order inside a class does not change a result: tiles are independent
        each([&](int b, int s, int i) {
            list[atomicAdd(&bin[b], 1)] = int2{s, i};
        });
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

// Loads 32 rows of one head of a tensor into LDS as float32, zeros past the
// sequence's last row and past dim. Lanes run along whichever of rows and
// features is consecutive in memory.
template <class IO, int DP>
__device__ __forceinline__ void load_rows(const AttnIo& x, int64_t at, int live, int dim,
                                          float (*to)[DP + 1]) {
    const bool rows_first = x.sr == 1 && x.sd != 1;
    for (int i = threadIdx.x; i < 32 * DP; i += kAttnThreads) {
        const int r = rows_first ? i % 32 : i / DP, f = rows_first ? i / 32 : i % DP;
        to[r][f] = r < live && f < dim ? IO::load(x.p, at + r * x.sr + f * x.sd) : 0.0f;
    }
}

// Packs 32 rows of one head: blockIdx.x the block of padded rows, blockIdx.y the
// head of an operand. With o given (dO and O) also delta, and dO's part only if
// it is packed.
template <bool SPLIT, int DP, class IO>
__global__ __launch_bounds__(kAttnThreads) void attn_pack_kernel(const AttnPack a) {
    __shared__ float x[32][DP + 1];
    __shared__ int32_t top;
    int which = 0, head = blockIdx.y;
    while (head >= a.op[which].heads) head -= a.op[which++].heads;
    const AttnPackOp& op = a.op[which];
    const int64_t padded = static_cast<int64_t>(blockIdx.x) * 32;
    if (padded >= op.rows) return;
    const RowOf ro = row_of(a.plan, op.keys, padded);
    if (!ro.any) return;
    const int n = op.keys ? ro.seq.nk : ro.seq.nq, first = op.keys ? ro.seq.k0 : ro.seq.q0;
    const int live = min(max(n - ro.row, 0), 32);
    const int64_t row = first + ro.row;
    if (threadIdx.x == 0) top = 0;
    load_rows<IO, DP>(op.src, ro.sid * op.src.sb + row * op.src.sr + head * op.src.sh, live,
                      a.dim, x);
    __syncthreads();

    if (a.delta != nullptr && which == 0) {
        // eight threads a row
        const int r = threadIdx.x / 8, part = threadIdx.x % 8;
        float d = 0.0f;
        const int64_t at = ro.sid * a.o.sb + (row + r) * a.o.sr + head * a.o.sh;
        if (r < live)
            for (int f = part; f < a.dim; f += 8)
                d = __builtin_fmaf(x[r][f], IO::load(a.o.p, at + f * a.o.sd), d);
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) d += __shfl_xor(d, s);
        if (part == 0) a.delta[head * a.delta_sh + padded + r] = r < live ? d : 0.0f;
        if constexpr (SPLIT) {
            const uint32_t bits = __float_as_uint(d) & 0x7fffffffu;
            if (part == 0 && r < live && bits < 0x7f800000u) atomicMax(&top, static_cast<int>(bits));
            __syncthreads();
            if (threadIdx.x == 0) {
                a.dexps[head * op.exps_sh + padded / 32] =
                    max(static_cast<int>(static_cast<uint32_t>(top) >> 23) - 127, -100);
                top = 0;
            }
            __syncthreads();
        }
    }
    if (op.dst == nullptr) return;

    float factor = 1.0f;
    if constexpr (SPLIT) {
        uint32_t m = 0;  // the largest finite magnitude
        for (int i = threadIdx.x; i < 32 * DP; i += kAttnThreads) {
            const uint32_t b = __float_as_uint(x[i / DP][i % DP]) & 0x7fffffffu;
            if (b < 0x7f800000u) m = max(m, b);
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(m, s)));
        if ((threadIdx.x & 63) == 0) atomicMax(&top, static_cast<int>(m));
        __syncthreads();
        const int e = max(static_cast<int>(static_cast<uint32_t>(top) >> 23) - 127, -100);
        factor = ldexpf(1.0f, kAttnUnit - e);
        if (threadIdx.x == 0) op.exps[head * op.exps_sh + padded / 32] = e;
    }
    constexpr int kPieces = DP / 8;
    char* const to = op.dst + head * op.dst_sh + padded * op.dst_sr;
    for (int i = threadIdx.x; i < 32 * kPieces; i += kAttnThreads) {
        const int r = i / kPieces, c = i % kPieces;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[r][8 * c + j] * factor;
        const AttnPair<SPLIT> f = attn_operand<SPLIT>(v);
        *reinterpret_cast<AttnFrag<SPLIT>*>(to + r * op.dst_sr + 16 * c) = f.f[0];
        if constexpr (SPLIT)
            *reinterpret_cast<AttnFrag<SPLIT>*>(to + r * op.dst_sr + 2 * DP + 16 * c) = f.f[1];
    }
}

template <bool SPLIT, class IO>
int pack(const AttnPack& a, int db, dim3 grid, hipStream_t st) {
    const dim3 wg(kAttnThreads);
    if (db == 1) hipLaunchKernelGGL((attn_pack_kernel<SPLIT, 32, IO>), grid, wg, 0, st, a);
    else if (db == 2) hipLaunchKernelGGL((attn_pack_kernel<SPLIT, 64, IO>), grid, wg, 0, st, a);
    else hipLaunchKernelGGL((attn_pack_kernel<SPLIT, 128, IO>), grid, wg, 0, st, a);
    return check_launch("attention: pack");
}

}  // namespace

int attn_launch_plan(const AttnPlanArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(attn_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    return check_launch("attention: plan");
}

int attn_launch_pack(const AttnPack& a, bool split, int db, int dtype, hipStream_t st) {
    int64_t rows = 0, heads = 0;
    for (int i = 0; i < a.n; ++i) {
        rows = rows > a.op[i].rows ? rows : a.op[i].rows;
        heads += a.op[i].heads;
    }
    if (rows == 0 || heads == 0) return SLK_OK;
    if (heads > 65535) return fail(SLK_EINVAL, "attention: too many heads");
    const dim3 grid(static_cast<unsigned>(rows / 32), static_cast<unsigned>(heads));
    if (dtype == SLK_F32) return pack<true, F32>(a, db, grid, st);
    (void)split;
    return pack<false, BF16>(a, db, grid, st);
}

}  // namespace slk
