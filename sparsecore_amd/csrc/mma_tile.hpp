// Matrix-core product of two packed operands, C = A·Bᵀ, with the epilogue as a
// functor: the loop behind the head and its loss (linear_ce.hip).
//
// Packed operand: R rows of K elements as stages of 128 bytes a row, stage by
// stage: P[stage][row][128 bytes], zero beyond K. A tile's stage is then one
// contiguous piece of memory, whatever K is. A stage holds, of a row,
//   SPLIT   32 elements in float16, high parts (64 bytes) then low parts: a
//           float32 x, scaled by a power of two, as hi + lo. The product takes
//           hi·hi + hi·lo + lo·hi in float32: x is kept to 2^-22 of itself (or
//           2^-39 of its row's largest element), about float32's own
//           rounding, at a third of the float16 rate, where the matrix cores'
//           float32 instructions run at a sixteenth;
//   else    64 elements in bfloat16.
// An operand is used along its stages (K inside a row) or across its rows: the
// same memory with K as the row and a stage as a panel of 32 (64) rows of the
// product ("turned" below). Turned fragments come out of LDS through the
// transposing read: a lane of each 16 names four columns of one of four rows and
// gets one column of all four. So every operand is packed once, whichever of the
// three products reads it.
//
// Tile: 256 x 128, eight waves of 64 x 64 (2 x 2 blocks of 32 x 32). Stages go
// from memory straight into a ring of three LDS buffers of 48 KiB, two stages
// ahead, one barrier a stage; the 16-byte pieces of a staged row are permuted
// (piece c of row r at slot c ^ ((r >> 1) & 7)), so that the 16 lanes of an
// LDS pass meet all banks once. Each buffer is an LDS variable of its own, named
// by a compile-time constant (the loop is unrolled by three): otherwise the
// compiler makes an LDS read wait for the loads just issued into another buffer.
#pragma once

#include "common.hpp"

namespace slk {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

constexpr int kStageBytes = 128;
template <bool SPLIT>
constexpr int kStageK = SPLIT ? 32 : 64;

constexpr int kTileM = 256, kTileN = 128;
constexpr int kMmaThreads = 512;
constexpr int kMmaBufs = 3;
constexpr int kMmaGroup = 4;  // tile rows of a group of the tile order

// s_waitcnt operand: at most n vector-memory loads outstanding, no LDS reads
// or scalar loads outstanding (n <= 63)
constexpr int wait_vm(int n) { return (n & 0xf) | ((n >> 4) << 14) | (0x7 << 4) | (0x0 << 8); }

// Which dimension is the device-side count of live tokens.
enum MmaLive { kLiveNone = 0, kLiveM = 1, kLiveN = 2, kLiveK = 3 };

// A turned operand's rows run along K: whole stages of them are there, zero (or
// finite, against zeros) where K ends inside one.
struct MmaArgs {
    const void* A;
    const void* B;
    int64_t M, N, nst;       // rows of A and B, stages (upper bounds where live says so)
    int64_t rows_a, rows_b;  // rows that the packed operands are laid out for
    const int32_t* live;
    int which;               // MmaLive
    int splits;              // parts of the K loop, each a workgroup of its own
};

// What an epilogue gets: its wave's NA x 2 blocks of 32 x 32 of a tile of
// 256 x BN. Lane l, register r of block [a][b]:
//   row  m0 + 32 a + 8 (r / 4) + 4 (l / 32) + r % 4,  column  n0 + 32 b + l % 32.
template <int NA, int BN>
struct MmaTile {
    static constexpr int kNA = NA, kBN = BN, kWavesM = kTileM / (32 * NA);
    int64_t i0, k0;  // the workgroup's tile
    int wm, wn, lane;
    int64_t M, N;
    int split;
    char* lds;  // a buffer of the ring (at least 48 KiB), free after a barrier
    __device__ __forceinline__ int64_t m0() const { return i0 + 32 * NA * wm; }
    __device__ __forceinline__ int64_t n0() const { return k0 + 64 * wn; }
    __device__ __forceinline__ int row(int a, int r) const {
        return 32 * a + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
    }
    __device__ __forceinline__ int col(int b) const { return 32 * b + (lane & 31); }
};

// The direct loads of a wave for an operand's stage of 64·PER rows (or of that
// many panel rows): load i = wv + 8 q fills lines 8 i .. 8 i + 7 of 128 bytes of
// the operand's buffer, lane l piece l mod 8 of line 8 i + l / 8. Pieces are
// permuted so that the lanes that read together meet all banks once: along the
// stage by the row, turned by rows 2, 3 of every four and by rows 4 to 7. A load
// is a scalar base (64 rows, or a panel; past the end the last one again) and
// one lane offset for all of them: an offset a load spilled registers.
template <bool SPLIT, bool TURN, int PER>
struct Loads {
    static constexpr int K = kStageK<SPLIT>;
    const char* base[PER];
    uint32_t off;
    int64_t step;
    __device__ __forceinline__ Loads(const void* P, int64_t R, int64_t limit, int64_t r0, int wv,
                                     int lane) {
        step = (TURN ? K : R) * kStageBytes;
        const int line = 8 * wv + lane / 8;
        off = TURN ? line % K * kStageBytes +
                         16 * ((lane & 7) ^ (4 * ((line >> 1) & 1) + 2 * ((line >> 2) & 1)))
                   : line * kStageBytes + 16 * ((lane & 7) ^ ((line >> 1) & 7));
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            constexpr int unit = TURN ? K : 64;
            const int64_t units = ceil_div(limit, unit);
            int64_t u = r0 / unit + (TURN ? 8 * (wv + 8 * q) / K : q);
            if (u >= units) u = units - 1;
            base[q] = static_cast<const char*>(P) + u * (TURN ? R : 64) * kStageBytes;
        }
    }
    __device__ __forceinline__ void issue(unsigned char* to, int wv, int64_t st) const {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass emits no stub of a kernel that calls this
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const uint64_t at = reinterpret_cast<uint64_t>(base[q] + st * step);
            const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
            const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
            const char* from =
                reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
            uint32_t o = off;
            asm("" : "+v"(o));  // keeps their sum with the load, whose own it is
            __builtin_amdgcn_global_load_lds(from + o, to + 1024 * (wv + 8 * q), 16, 0, 0);
        }
#endif
    }
};

typedef short i16x4 __attribute__((ext_vector_type(4)));

// The transposing LDS read: each lane of 16 names four 16-bit elements; lane l
// gets element l % 4 of what lanes l / 4, 4 + l / 4, 8 + l / 4, 12 + l / 4 named.
__device__ __forceinline__ i16x4 read_turned(const unsigned char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    using Piece = __attribute__((address_space(3))) i16x4*;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((Piece)(const_cast<unsigned char*>(lds)));
#else
    (void)lds;  // the host pass has no LDS
    return i16x4{};
#endif
}

// Fragments of the operand's 32-row blocks from a staged buffer: block `b` of
// the wave's rows (first row r0 of the tile), k-step ks, part 0 (high or only)
// or 1 (low). Lane l gets row l % 32, K 16 ks + 8 (l / 32) ...
template <bool SPLIT, bool TURN>
struct Frags {
    using Frag = std::conditional_t<SPLIT, f16x8, b16x8>;
    static constexpr int K = kStageK<SPLIT>;
    int row, half;    // along the stage
    int at[2][2];     // turned: byte of [part, or odd block][four rows of eight]
    __device__ __forceinline__ Frags(int r0, int lane) {
        half = lane >> 5;
        row = r0 + (lane & 31);
        const int i = lane & 15, ch = (lane >> 4) & 1;
        // row r0 is the first of a panel: 32 rows of a split operand, 64 of the other
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int piece = (4 * p + 2 * ch + ((i >> 1) & 1)) ^ (4 * ((i >> 3) & 1) + 2 * h);
                at[p][h] = (r0 / K * K + 8 * half + 4 * h + (i >> 2)) * kStageBytes + 16 * piece +
                           8 * (i & 1);
            }
    }
    __device__ __forceinline__ Frag read(const unsigned char* buf, int b, int ks, int part) const {
        if constexpr (TURN) {
            const int p = SPLIT ? part : b & 1, panel = SPLIT ? b : b >> 1;
            const int o = (panel * K + 16 * ks) * kStageBytes;
            const i16x4 lo = read_turned(buf + at[p][0] + o);
            const i16x4 hi = read_turned(buf + at[p][1] + o);
            return __builtin_bit_cast(Frag,
                                      __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int r = row + 32 * b, c = (SPLIT ? 4 * part : 0) + 2 * ks + half;
            return *reinterpret_cast<const Frag*>(buf + 16 * (r * 8 + (c ^ ((r >> 1) & 7))));
        }
    }
};

// A workgroup's tile and part of the K loop. Grouped, XCD-contiguous tile order:
// consecutive tiles share rows of A and B. The launch keeps tiles x splits under
// 2^31, so that the divisions take 32 bits; the results are put back into scalar
// registers, which the loads' bases come from.
struct MmaWork {
    int64_t M, N, i0, k0, s0, s1;
    int split;
    bool any;  // false for the whole workgroup: past the live tiles
    template <int K, int TN>
    static __device__ __forceinline__ MmaWork of(const MmaArgs& g) {
        MmaWork w;
        w.M = g.M;
        w.N = g.N;
        int64_t nst = g.nst;
        if (g.which != kLiveNone) {
            const int64_t live = *g.live;
            if (g.which == kLiveM) w.M = live;
            else if (g.which == kLiveN) w.N = live;
            else nst = ceil_div(live, K);
        }
        const uint32_t nTi = static_cast<uint32_t>(ceil_div(w.M, kTileM));
        const uint32_t nTk = static_cast<uint32_t>(ceil_div(w.N, TN));
        const uint32_t tiles = nTi * nTk, splits = g.splits, total = tiles * splits;
        w.any = blockIdx.x < total;
        if (!w.any) return w;
        const uint32_t L = static_cast<uint32_t>(xcd_logical_block(blockIdx.x, total));
        const uint32_t split = splits > 1 ? L / tiles : 0;
        const uint32_t tile = L - split * tiles;
        const uint32_t grp = tile / (kMmaGroup * nTk);
        const uint32_t first = grp * kMmaGroup;
        const uint32_t gsize = nTi - first < kMmaGroup ? nTi - first : kMmaGroup;
        const uint32_t in_grp = tile - grp * kMmaGroup * nTk;
        const uint32_t col = in_grp / gsize;
        const uint32_t per = static_cast<uint32_t>(nst) / splits;
        const uint32_t extra = static_cast<uint32_t>(nst) % splits;
        auto uniform = [](uint32_t x) {
            return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
        };
        w.i0 = uniform(first + in_grp - col * gsize) * kTileM;
        w.k0 = uniform(col) * TN;
        w.split = static_cast<int>(uniform(split));
        w.s0 = uniform(split * per + (split < extra ? split : extra));
        w.s1 = uniform(split * per + per + (split < extra ? split + 1 : extra));
        return w;
    }
};

template <bool SPLIT, bool TA, bool TB, class Epi>
__global__ __launch_bounds__(kMmaThreads) void mma_kernel(const MmaArgs g, const Epi epi) {
    __shared__ __align__(16) unsigned char ring0[(kTileM + kTileN) * kStageBytes];
    __shared__ __align__(16) unsigned char ring1[(kTileM + kTileN) * kStageBytes];
    __shared__ __align__(16) unsigned char ring2[(kTileM + kTileN) * kStageBytes];

    const MmaWork w = MmaWork::of<kStageK<SPLIT>, kTileN>(g);
    if (!w.any) return;
    const int64_t M = w.M, N = w.N, i0 = w.i0, k0 = w.k0, s0 = w.s0, s1 = w.s1;
    const int split = w.split;

    const int t = threadIdx.x;
    const int lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wv >> 1, wn = wv & 1;

    constexpr int kPerA = kTileM / 64, kPerB = kTileN / 64;
    const Loads<SPLIT, TA, kPerA> la(g.A, g.rows_a, M, i0, wv, lane);
    const Loads<SPLIT, TB, kPerB> lb(g.B, g.rows_b, N, k0, wv, lane);
    auto issue = [&](int buf, int64_t st) {
        unsigned char* to = buf == 0 ? ring0 : buf == 1 ? ring1 : ring2;
        la.issue(to, wv, st);
        lb.issue(to + kTileM * kStageBytes, wv, st);
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.0f;

    const Frags<SPLIT, TA> fa(wm * 64, lane);
    const Frags<SPLIT, TB> fb(wn * 64, lane);
    // fragments of half a stage: SPLIT, a k-step's high and low parts; else two k-steps
    typename Frags<SPLIT, TA>::Frag af[2][2][2], bf[2][2][2];  // [half stage][block][part]
    auto reads = [&](const unsigned char* buf, int h) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int ks = SPLIT ? h : 2 * h + p, part = SPLIT ? p : 0;
                af[h][b][p] = fa.read(buf, b, ks, part);
                bf[h][b][p] = fb.read(buf + kTileM * kStageBytes, b, ks, part);
            }
    };
    auto mfmas = [&](int h, int pa, int pb) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if constexpr (SPLIT) {
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[h][a][pa], bf[h][b][pb],
                                                                       acc[a][b], 0, 0, 0);
                } else {
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        af[h][a][pa], bf[h][b][pb], acc[a][b], 0, 0, 0);
                }
            }
    };
    constexpr int kLoads = kPerA + kPerB;
    // Stage st reads buffer st mod 3 and loads stage st + 2 into the buffer that
    // stage st - 1 left. The barrier sits after the stage's last LDS reads: by
    // then this wave's loads of stage st + 1 have landed (its loads of stage
    // st + 2 may be in flight), so behind it every wave's have, and the buffer
    // of stage st is free. A bare s_barrier: __syncthreads would also wait for
    // the loads of stage st + 2. Past the end the last stage is loaded again,
    // so that every stage waits for the same count.
    auto stage = [&](auto I, int64_t st) {
        constexpr int buf = decltype(I)::value;
        mfmas(0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        reads(buf == 0 ? ring0 : buf == 1 ? ring1 : ring2, 1);
        issue((buf + 2) % kMmaBufs, st + 2 < s1 ? st + 2 : s1 - 1);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (SPLIT) {
            mfmas(0, 0, 1);
            mfmas(0, 1, 0);
        } else {
            mfmas(0, 1, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(wait_vm(kLoads));
        asm volatile("s_barrier" ::: "memory");
        reads(buf == 0 ? ring1 : buf == 1 ? ring2 : ring0, 0);
        __builtin_amdgcn_sched_barrier(0);
        mfmas(1, 0, 0);
        if constexpr (SPLIT) {
            mfmas(1, 0, 1);
            mfmas(1, 1, 0);
        } else {
            mfmas(1, 1, 1);
        }
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    using B2 = std::integral_constant<int, 2>;
    if (s0 < s1) {
        issue(0, s0);
        issue(1, s0 + 1 < s1 ? s0 + 1 : s0);
        __builtin_amdgcn_s_waitcnt(wait_vm(kLoads));
        asm volatile("s_barrier" ::: "memory");
        reads(ring0, 0);
        int64_t st = s0;
        for (; st + 3 <= s1; st += 3) {
            stage(B0{}, st);
            stage(B1{}, st + 1);
            stage(B2{}, st + 2);
        }
        if (st < s1) stage(B0{}, st);
        if (st + 1 < s1) stage(B1{}, st + 1);
        __builtin_amdgcn_s_waitcnt(0);  // no direct load still writing LDS
    }
    epi(acc, MmaTile<2, kTileN>{i0, k0, wm, wn, lane, M, N, split,
                                reinterpret_cast<char*>(ring0)});
}

// The same product in tiles of 256 x 256: eight waves of 128 x 64 (2 x 4), a
// ring of two stages of 64 KiB. A wave reads six fragments for eight
// instructions (24 of a split operand's), where the smaller tile reads eight
// for eight: with one a stage of the bfloat16 product kept the LDS busy for
// 1408 cycles (reads, and the direct loads' writes) against 1024 of the matrix
// cores, now for 2048 against 2048. Fragments are read one k-step ahead. The
// barrier sits before a stage's last k-step, whose fragments are in registers:
// every wave has read the stage, and its loads of the next have landed; the
// stage's buffer is then filled with the stage after the next, a whole stage's
// time before that is read.
constexpr int kWideN = 256;

template <bool SPLIT, bool TA, bool TB, class Epi>
__global__ __launch_bounds__(kMmaThreads) void mma_wide_kernel(const MmaArgs g, const Epi epi) {
    __shared__ __align__(16) unsigned char ring0[(kTileM + kWideN) * kStageBytes];
    __shared__ __align__(16) unsigned char ring1[(kTileM + kWideN) * kStageBytes];

    const MmaWork w = MmaWork::of<kStageK<SPLIT>, kWideN>(g);
    if (!w.any) return;
    const int64_t M = w.M, N = w.N, i0 = w.i0, k0 = w.k0, s0 = w.s0, s1 = w.s1;
    const int split = w.split;

    const int t = threadIdx.x;
    const int lane = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wv >> 2, wn = wv & 3;

    constexpr int kPer = kTileM / 64;  // loads of a wave and stage, of each operand
    const Loads<SPLIT, TA, kPer> la(g.A, g.rows_a, M, i0, wv, lane);
    const Loads<SPLIT, TB, kPer> lb(g.B, g.rows_b, N, k0, wv, lane);
    auto issue = [&](int buf, int64_t st) {
        unsigned char* to = buf ? ring1 : ring0;
        la.issue(to, wv, st);
        lb.issue(to + kTileM * kStageBytes, wv, st);
    };

    f32x16 acc[4][2];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.0f;

    const Frags<SPLIT, TA> fa(wm * 128, lane);
    const Frags<SPLIT, TB> fb(wn * 64, lane);
    // [set][block]; a set is a k-step's parity, or (SPLIT) 0: high parts, 1: low parts
    typename Frags<SPLIT, TA>::Frag af[2][4], bf[2][2];
    // k-step ks of A's rows (first two, last two blocks) and of B's, into a set
    auto read_a = [&](const unsigned char* buf, int ks, int set, int a0) {
#pragma unroll
        for (int a = a0; a < a0 + 2; ++a) af[set][a] = fa.read(buf, a, ks, SPLIT ? set : 0);
    };
    auto read_b = [&](const unsigned char* buf, int ks, int set) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
            bf[set][b] = fb.read(buf + kTileM * kStageBytes, b, ks, SPLIT ? set : 0);
    };
    auto mfmas = [&](int a, int sa, int sb) {  // one row of blocks
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if constexpr (SPLIT) {
                acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[sa][a], bf[sb][b], acc[a][b],
                                                                   0, 0, 0);
            } else {
                acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[sa][a], bf[sb][b],
                                                                    acc[a][b], 0, 0, 0);
            }
        }
    };
    // Eight instructions with other work between them: the matrix cores take 32
    // cycles each, during which the wave issues the work. The reads that they
    // use were issued eight instructions ago, so the wait before them is free.
    auto eight = [&](int sa, int sb, auto&& w0, auto&& w1, auto&& w2) {
        __builtin_amdgcn_s_waitcnt(wait_vm(63));
        __builtin_amdgcn_sched_barrier(0);
        mfmas(0, sa, sb);
        __builtin_amdgcn_sched_barrier(0);
        w0();
        __builtin_amdgcn_sched_barrier(0);
        mfmas(1, sa, sb);
        __builtin_amdgcn_sched_barrier(0);
        w1();
        __builtin_amdgcn_sched_barrier(0);
        mfmas(2, sa, sb);
        __builtin_amdgcn_sched_barrier(0);
        w2();
        __builtin_amdgcn_sched_barrier(0);
        mfmas(3, sa, sb);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto none = [] {};
    auto meet = [&] {
        __builtin_amdgcn_s_waitcnt(wait_vm(0));
        asm volatile("s_barrier" ::: "memory");
    };
    // A k-step's fragments ahead of its instructions: all of the next k-step's
    // (bfloat16); of a split operand the part whose registers the last eight
    // instructions freed (the order lo·hi, hi·hi, hi·lo makes that three groups).
    auto stage = [&](auto I, int64_t st) {
        constexpr int buf = decltype(I)::value;
        const unsigned char* cur = buf ? ring1 : ring0;
        const unsigned char* nxt = (buf ? ring0 : ring1);
        // past the end the last stage is loaded again, unused
        const int64_t ahead = st + 2 < s1 ? st + 2 : s1 - 1;
        if constexpr (SPLIT) {
            eight(1, 0, [&] { read_a(cur, 0, 0, 0); }, [&] { read_a(cur, 0, 0, 2); },
                  [&] { read_b(cur, 0, 1); });
            eight(0, 0, [&] { read_a(cur, 1, 1, 0); }, [&] { read_a(cur, 1, 1, 2); }, none);
            eight(0, 1, [&] { read_b(cur, 1, 0); }, none, none);
            eight(1, 0, [&] { read_a(cur, 1, 0, 0); }, [&] { read_a(cur, 1, 0, 2); },
                  [&] { read_b(cur, 1, 1); });
            meet();
            eight(0, 0, [&] { read_a(nxt, 0, 1, 0); },
                  [&] { read_a(nxt, 0, 1, 2); }, [&] { issue(buf, ahead); });
            eight(0, 1, [&] { read_b(nxt, 0, 0); }, none, none);
        } else {
#pragma unroll
            for (int ks = 0; ks < 3; ++ks) {
                const int set = (ks + 1) & 1;
                eight(ks & 1, ks & 1, [&] { read_b(cur, ks + 1, set); },
                      [&] { read_a(cur, ks + 1, set, 0); }, [&] { read_a(cur, ks + 1, set, 2); });
            }
            meet();
            eight(1, 1, [&] { read_b(nxt, 0, 0); read_a(nxt, 0, 0, 0); },
                  [&] { read_a(nxt, 0, 0, 2); }, [&] { issue(buf, ahead); });
        }
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    if (s0 < s1) {
        issue(0, s0);
        issue(1, s0 + 1 < s1 ? s0 + 1 : s0);
        __builtin_amdgcn_s_waitcnt(wait_vm(2 * kPer));
        asm volatile("s_barrier" ::: "memory");
        read_a(ring0, 0, SPLIT ? 1 : 0, 0);
        read_a(ring0, 0, SPLIT ? 1 : 0, 2);
        read_b(ring0, 0, 0);
        int64_t st = s0;
        for (; st + 2 <= s1; st += 2) {
            stage(B0{}, st);
            stage(B1{}, st + 1);
        }
        if (st < s1) stage(B0{}, st);
        __builtin_amdgcn_s_waitcnt(0);  // no direct load still writing LDS
    }
    epi(acc, MmaTile<4, kWideN>{i0, k0, wm, wn, lane, M, N, split,
                                reinterpret_cast<char*>(ring0)});
}

// Wide tiles where their rounds on the card's 256 CUs take no longer: a wide stage
// takes about 1.7 times a small one's.
inline bool mma_wide(int64_t M, int64_t N, int splits) {
    const int64_t small = ceil_div(ceil_div(M, kTileM) * ceil_div(N, kTileN) * splits, 256);
    const int64_t wide = ceil_div(ceil_div(M, kTileM) * ceil_div(N, kWideN) * splits, 256);
    return 17 * wide <= 10 * small;
}

// Rounds of 256 workgroups that a product takes, in small tiles' time.
inline double mma_rounds(int64_t M, int64_t N) {
    const bool wide = mma_wide(M, N, 1);
    const int64_t tiles = ceil_div(M, kTileM) * ceil_div(N, wide ? kWideN : kTileN);
    return static_cast<double>(ceil_div(tiles, 256)) * (wide ? 1.7 : 1.0);
}

// Launches C = A·Bᵀ over an upper bound of its tiles. The two widths add the terms of
// a stage in different orders: a product that has to repeat another's bits names its
// width.
template <bool SPLIT, bool TA, bool TB, class Epi>
int mma(const MmaArgs& g, const Epi& epi, hipStream_t st, const char* who, bool wide) {
    const int64_t groups =
        ceil_div(g.M, kTileM) * ceil_div(g.N, wide ? kWideN : kTileN) * g.splits;
    if (groups == 0) return SLK_OK;
    if (groups > max_groups(kMmaThreads)) {
        return fail(SLK_EINVAL, std::string(who) + ": too many tiles");
    }
    const dim3 grid(static_cast<unsigned>(groups)), wg(kMmaThreads);
    if (wide) hipLaunchKernelGGL((mma_wide_kernel<SPLIT, TA, TB, Epi>), grid, wg, 0, st, g, epi);
    else hipLaunchKernelGGL((mma_kernel<SPLIT, TA, TB, Epi>), grid, wg, 0, st, g, epi);
    return check_launch(who);
}

template <bool SPLIT, bool TA, bool TB, class Epi>
int mma(const MmaArgs& g, const Epi& epi, hipStream_t st, const char* who) {
    return mma<SPLIT, TA, TB>(g, epi, st, who, mma_wide(g.M, g.N, g.splits));
}

}  // namespace slk
