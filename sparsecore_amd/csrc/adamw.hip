// AdamW over many tensors at once, moments in 32 or in 8 bits, and the moves
// of moments that follow a padded-CSR topology rewrite.
//
//   m = b1·m + (1 - b1)·g        v = b2·v + (1 - b2)·g²
//   p = (1 - lr·wd)·p - lr / (1 - b1^t) · m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A step moves 28 bytes an element with float32 parameters and moments, 16
// with 8-bit moments, for some fifteen operations: it is bound by memory, and
// for a small model by the launch. So the tensors' table travels as a kernel
// argument (no copy to the device, nothing to keep alive) and one launch
// serves kAdamTensors tensors; a lane takes four consecutive elements with
// one 16-byte load an array; a wave takes SLK_Q8_BLOCK elements, a whole
// block of 8-bit codes, whose new scale is one wave reduction. Measured: 64
// million elements with 8-bit moments 217 us (4.7 TB/s, what a large copy
// reaches), 53 tensors of 2.3 million with 32-bit ones 11.4 us (out of the
// caches), 49 thousand elements 3.8 us.
#include "elem.hpp"
#include "q8.hpp"

namespace slk {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kAdamTensors = 56;  // tensors of one launch: the argument stays below 4 KiB
constexpr int kAdamWaves = kAdamThreads / kWave;
constexpr int kAdamSpan = kAdamWaves * kQ8Block;  // elements of one workgroup

struct AdamTable {
    slk_adamw_tensor t[kAdamTensors];
    uint32_t first[kAdamTensors];  // first workgroup of each tensor
    int32_t n;
    uint64_t aligned;  // bit i: tensor i's arrays take four elements a load
};

struct AdamCoef {
    float b1, omb1, b2, omb2, eps;
    float decay, step_size, inv_root;  // 1 - lr·wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    // where the step or the learning rate lives on the device:
    const float* step;
    const float* lr;
    double lr_host, wd, log_b1, log_b2, step_host;
};

// four codes of a block: element i, i + 1, i + 2, i + 3 (those below n)
template <bool SIGNED>
__device__ __forceinline__ void decode4(const void* codes, int64_t i, int64_t n, bool vec,
                                        float scale, float (&v)[4]) {
    uint32_t w = 0;
    const uint8_t* c = static_cast<const uint8_t*>(codes);
    if (vec) {
        w = *reinterpret_cast<const uint32_t*>(c + i);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) w |= static_cast<uint32_t>(c[i + j]) << (8 * j);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t b = (w >> (8 * j)) & 0xffu;
        v[j] = SIGNED ? q8_decode_signed(static_cast<int8_t>(b), scale)
                      : q8_decode_unsigned(static_cast<int>(b), scale);
    }
}

template <bool SIGNED>
__device__ __forceinline__ void encode4(void* codes, int64_t i, int64_t n, bool vec, float scale,
                                        const float (&v)[4]) {
    uint32_t w = 0;
    const float rcp = q8_reciprocal(scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int q = SIGNED ? q8_encode_signed(v[j], scale, rcp)
                             : q8_encode_unsigned(v[j], scale, rcp);
        w |= (static_cast<uint32_t>(q) & 0xffu) << (8 * j);
    }
    uint8_t* c = static_cast<uint8_t*>(codes);
    if (vec) {
        *reinterpret_cast<uint32_t*>(c + i) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) c[i + j] = static_cast<uint8_t>(w >> (8 * j));
    }
}

template <class T>
__device__ __forceinline__ void load_some(const void* p, int64_t i, int64_t n, bool vec,
                                          float (&v)[4]) {
    if (vec) {
        T::load4(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j < n ? T::load(p, i + j) : 0.0f;
    }
}

template <class T>
__device__ __forceinline__ void store_some(void* p, int64_t i, int64_t n, bool vec,
                                           const float (&v)[4]) {
    if (vec) {
        T::store4(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) T::store(p, i + j, v[j]);
    }
}

template <class T, bool Q8>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(const AdamTable tab,
                                                             const AdamCoef c) {
    // the tensor of this workgroup: the last whose first workgroup is not past it
    int lo = 0, hi = tab.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const slk_adamw_tensor& t = tab.t[lo];
    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t block = static_cast<int64_t>(blockIdx.x - tab.first[lo]) * kAdamWaves + wv;
    const int64_t i = block * kQ8Block + 4 * lane;
    if (block * kQ8Block >= t.n) return;  // whole waves; there is no barrier below
    const bool vec = ((tab.aligned >> lo) & 1u) && i + 4 <= t.n;

    float decay = c.decay, step_size = c.step_size, inv_root = c.inv_root;
    if (c.step != nullptr || c.lr != nullptr) {
        const double step = c.step != nullptr ? static_cast<double>(*c.step) : c.step_host;
        const double lr = c.lr != nullptr ? static_cast<double>(*c.lr) : c.lr_host;
        decay = static_cast<float>(1.0 - lr * c.wd);
        step_size = static_cast<float>(lr / -expm1(step * c.log_b1));
        inv_root = static_cast<float>(1.0 / sqrt(-expm1(step * c.log_b2)));
    }

    float p[4], g[4], m[4], v[4];
    load_some<T>(t.param, i, t.n, vec, p);
    load_some<T>(t.grad, i, t.n, vec, g);
    if (Q8) {
        decode4<true>(t.exp_avg, i, t.n, vec, t.exp_avg_scale[block], m);
        decode4<false>(t.exp_avg_sq, i, t.n, vec, t.exp_avg_sq_scale[block], v);
    } else {
        load_some<F32>(t.exp_avg, i, t.n, vec, m);
        load_some<F32>(t.exp_avg_sq, i, t.n, vec, v);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = c.b1 * m[j] + c.omb1 * g[j];
        v[j] = c.b2 * v[j] + c.omb2 * (g[j] * g[j]);
        // the instructions' square root and reciprocal are within an ulp; the
        // root's takes no subnormals, so a tiny v is scaled by 2^64 around it
        const bool tiny = v[j] < 0x1p-96f;
        float root = __builtin_amdgcn_sqrtf(tiny ? v[j] * 0x1p64f : v[j]);
        root = (tiny ? root * 0x1p-32f : root) * inv_root + c.eps;
        p[j] = p[j] * decay - step_size * (m[j] * __builtin_amdgcn_rcpf(root));
    }
    store_some<T>(t.param, i, t.n, vec, p);
    if (Q8) {
        // elements past the tensor's end were read as 0 and stay 0
        const float ms = q8_block_max(m), vs = q8_block_max(v);
        encode4<true>(t.exp_avg, i, t.n, vec, ms, m);
        encode4<false>(t.exp_avg_sq, i, t.n, vec, vs, v);
        if (lane == 0) {
            t.exp_avg_scale[block] = ms;
            t.exp_avg_sq_scale[block] = vs;
        }
    } else {
        store_some<F32>(t.exp_avg, i, t.n, vec, m);
        store_some<F32>(t.exp_avg_sq, i, t.n, vec, v);
    }
}

template <bool SIGNED>
__global__ __launch_bounds__(kAdamThreads) void q8_decode_kernel(const void* __restrict__ codes,
                                                                 const float* __restrict__ scales,
                                                                 int64_t n, bool aligned,
                                                                 float* __restrict__ out) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * kAdamThreads + threadIdx.x) * 4;
    if (i >= n) return;
    const bool vec = aligned && i + 4 <= n;
    float v[4];
    decode4<SIGNED>(codes, i, n, vec, scales[i / kQ8Block], v);
    store_some<F32>(out, i, n, vec, v);
}

template <bool SIGNED>
__global__ __launch_bounds__(kAdamThreads) void q8_encode_kernel(const float* __restrict__ x,
                                                                 int64_t n, bool aligned,
                                                                 void* __restrict__ codes,
                                                                 float* __restrict__ scales) {
    const int64_t block = static_cast<int64_t>(blockIdx.x) * kAdamWaves + (threadIdx.x >> 6);
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t i = block * kQ8Block + 4 * lane;
    if (block * kQ8Block >= n) return;
    const bool vec = aligned && i + 4 <= n;
    float v[4];
    load_some<F32>(x, i, n, vec, v);
    const float s = q8_block_max(v);
    encode4<SIGNED>(codes, i, n, vec, s, v);
    if (lane == 0) scales[block] = s;
}

// ───────────────── moments that follow a topology rewrite ─────────────────

struct CarryTable {
    slk_carry_state s[SLK_CARRY_STATES];
    int32_t n;
};

// How many of row_start[lo, hi) are at most s, plus lo; all before lo are. The
// wave looks at 64 places at a time: three dependent loads for 16384 rows.
__device__ __forceinline__ int wave_rows_upto(const int32_t* __restrict__ row_start, int s, int lo,
                                              int hi, int lane) {
    while (lo < hi) {
        const int step = (hi - lo + kWave - 1) / kWave;
        // (lo + 63 step can pass int32 for two thousand million rows)
        const int64_t at = lo + static_cast<int64_t>(lane) * step;
        const int c = __popcll(__ballot(at < hi && row_start[at < hi ? at : lo] <= s));
        if (c == 0) break;
        const int64_t up = lo + static_cast<int64_t>(c) * step;
        lo += (c - 1) * step + 1;
        hi = up < hi ? static_cast<int>(up) : hi;
    }
    return lo;
}

// col's place among old_cols[lo, hi), ascending, or -1.
__device__ inline int find_slot(const int32_t* __restrict__ old_cols, int lo, int hi, int col) {
    const int stop = hi;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (old_cols[mid] < col) lo = mid + 1; else hi = mid;
    }
    return lo < stop && old_cols[lo] == col ? lo : -1;
}

// One thread per four slots, one wave per SLK_Q8_BLOCK slots. Each live slot
// of the new topology looks its column up among its row's old columns (both
// ascending) and takes that slot's state; a grown connection and padding take
// 0. Out of place: a row's slots move both ways.
//
// Bound by its instructions (16 million slots in 8 bits moved in 185 us when
// every slot searched its row by itself with 64-bit places, 153 now, where their
// bytes take 41), then by the latency of dependent loads. The wave finds its first row 64 places at a time
// and brings the old columns of its own slots and kNear on either side into
// LDS: a column is mostly that near to where it was (a rewrite that moves a
// third of a row of 16384 shifts the rest by about a hundred slots). A lane
// searches its first column of a row in ten steps without a branch and its next
// ones within seven places of the last; what these miss is searched in memory.
// Slots are below 2^31.
constexpr int kNear = 256, kWindow = kQ8Block + 2 * kNear;

__global__ __launch_bounds__(kAdamThreads) void carry_kernel(
    const int32_t* __restrict__ row_start, int nrows, int total,
    const int32_t* __restrict__ old_cols, const int32_t* __restrict__ old_nnz,
    const int32_t* __restrict__ new_cols, const int32_t* __restrict__ new_nnz,
    const CarryTable tab) {
    __shared__ int32_t windows[kAdamWaves][kWindow + 8];
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int block = static_cast<int>(blockIdx.x) * kAdamWaves + wv;
    const int lane = threadIdx.x & (kWave - 1);
    if (static_cast<int64_t>(block) * kQ8Block >= total) return;  // a wave; no barrier below
    const int first = block * kQ8Block;
    const int last = total - first > kQ8Block ? first + kQ8Block - 1 : total - 1;
    const int i = first + 4 * lane;  // below 2^31 + 256: compared as total - i

    int32_t* win = windows[wv];
    const int w0 = first > kNear ? first - kNear : 0;
    const int w1 = total - last > kNear ? last + 1 + kNear : total;
    int32_t col[4];
#pragma unroll
    for (int j = 0; j < kWindow / kWave; ++j) {
        const int at = j * kWave + lane;
        win[at] = at < w1 - w0 ? old_cols[w0 + at] : 0;
    }
    const int mine = 4 * lane;  // this lane's place among the wave's slots
#pragma unroll
    for (int j = 0; j < 4; ++j) col[j] = mine + j <= last - first ? new_cols[i + j] : -1;
    const int r0 = wave_rows_upto(row_start, first, 0, nrows, lane) - 1;
    // mostly the same row or one of the next few
    const int near = nrows - r0 > kWave + 1 ? r0 + 1 + kWave : nrows;
    int r1 = wave_rows_upto(row_start, last, r0 + 1, near, lane) - 1;
    if (r1 + 1 == near && near < nrows)
        r1 = wave_rows_upto(row_start, last, near, nrows, lane) - 1;

    // the lane's first row, its old columns [start, end), its live slots and its
    // old columns' part of the window
    int row = r0;
    if (r0 != r1) {
        const int s = mine <= last - first ? i : last;
        int lo = r0 + 1, hi = r1 + 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (row_start[mid] <= s) lo = mid + 1; else hi = mid;
        }
        row = lo - 1;
    }
    int start, end, live, next, lo, hi;
    auto enter = [&] {
        const int r = row >= 0 ? row : 0;
        start = row_start[r];
        live = start + (row >= 0 ? new_nnz[r] : 0) - first;
        next = (row + 1 < nrows ? row_start[row + 1] : total) - first;
        const int64_t old_end = static_cast<int64_t>(start) + (row >= 0 ? old_nnz[r] : 0);
        end = old_end < total ? static_cast<int>(old_end) : total;
        lo = (start > w0 ? start : w0) - w0;
        hi = (end < w1 ? end : w1) - w0;
    };
    enter();
    int from[4], pos = lo;
    bool fresh = true;  // pos says nothing about this row yet
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (mine + j >= next && mine + j <= last - first) {
            while (row < r1 && mine + j >= next) {
                ++row;
                next = (row + 1 < nrows ? row_start[row + 1] : total) - first;
            }
            enter();
            pos = lo;
            fresh = true;
        }
        auto step = [&](int b) {
            const int t = pos + b;
            const int at = t <= hi ? t - 1 : 0;
            pos = t <= hi && win[at] < col[j] ? t : pos;
        };
        if (__any(fresh)) {
#pragma unroll
            for (int b = 512; b > 4; b >>= 1) step(b);
        }
#pragma unroll
        for (int b = 4; b > 0; b >>= 1) step(b);
        if (!fresh) {
            while (pos < hi && win[pos] < col[j]) ++pos;
        }
        fresh = false;
        const bool wanted = mine + j < live && mine + j <= last - first;
        const bool in = lo < hi;
        from[j] = wanted && in && pos < hi && win[pos] == col[j] ? w0 + pos : -1;
        // not in the window: before it, behind it, or nowhere
        const bool before = wanted && from[j] < 0 && in && pos == lo && w0 + lo > start;
        const bool behind = wanted && from[j] < 0 && in && pos == hi && w0 + hi < end;
        if (before || behind || (wanted && !in && start < end)) {
            from[j] = find_slot(old_cols, behind ? w0 + hi : start, before ? w0 + lo : end, col[j]);
        }
    }

    // all states' loads first, then their stores
    const int64_t at = static_cast<int64_t>(first) + mine;
    float v[SLK_CARRY_STATES][4];
#pragma unroll
    for (int k = 0; k < SLK_CARRY_STATES; ++k) {
        if (k >= tab.n) break;
        const slk_carry_state& st = tab.s[k];
        if (st.kind == SLK_STATE_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[k][j] = from[j] >= 0 ? static_cast<const float*>(st.src)[from[j]] : 0.0f;
        } else {
            int q[4];
            float scale[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int f = from[j] >= 0 ? from[j] : 0;
                q[j] = static_cast<const uint8_t*>(st.src)[f];
                scale[j] = st.src_scale[f / kQ8Block];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = st.kind == SLK_STATE_Q8_SIGNED
                                    ? q8_decode_signed(static_cast<int8_t>(q[j]), scale[j])
                                    : q8_decode_unsigned(q[j], scale[j]);
                v[k][j] = from[j] >= 0 ? x : 0.0f;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < SLK_CARRY_STATES; ++k) {
        if (k >= tab.n) break;
        const slk_carry_state& st = tab.s[k];
        if (st.kind == SLK_STATE_F32) {
            const bool vec =
                total - first >= mine + 4 && (reinterpret_cast<uintptr_t>(st.dst) & 15) == 0;
            store_some<F32>(st.dst, at, total, vec, v[k]);
        } else {
            const bool vec =
                total - first >= mine + 4 && (reinterpret_cast<uintptr_t>(st.dst) & 3) == 0;
            const float scale = q8_block_max(v[k]);
            if (st.kind == SLK_STATE_Q8_SIGNED) encode4<true>(st.dst, at, total, vec, scale, v[k]);
            else encode4<false>(st.dst, at, total, vec, scale, v[k]);
            if (lane == 0) st.dst_scale[block] = scale;
        }
    }
}

}  // namespace
}  // namespace slk

extern "C" int slk_adamw(const slk_adamw_tensor* tensors_host, int64_t n_tensors, int dtype,
                         int state_bits, const slk_adamw_args* args_host, void* stream) {
    using namespace slk;
    clear_error();
    if (n_tensors < 0 || (n_tensors > 0 && tensors_host == nullptr) || args_host == nullptr) {
        return fail(SLK_EINVAL, "adamw: NULL table or a negative number of tensors");
    }
    if (dtype != SLK_F32 && dtype != SLK_BF16) {
        return fail(SLK_EINVAL, "adamw: dtype must be SLK_F32 or SLK_BF16");
    }
    if (state_bits != 8 && state_bits != 32) {
        return fail(SLK_EINVAL, "adamw: state_bits must be 8 or 32, got " +
                                    std::to_string(state_bits));
    }
    const slk_adamw_args& a = *args_host;
    if (!(a.beta1 >= 0.0 && a.beta1 < 1.0) || !(a.beta2 >= 0.0 && a.beta2 < 1.0)) {
        return fail(SLK_EINVAL, "adamw: betas must lie in [0, 1)");
    }
    if (a.step_dev == nullptr && !(a.step >= 1.0)) {
        return fail(SLK_EINVAL, "adamw: step must be at least 1");
    }
    AdamCoef c;
    c.b1 = static_cast<float>(a.beta1);
    c.omb1 = static_cast<float>(1.0 - a.beta1);
    c.b2 = static_cast<float>(a.beta2);
    c.omb2 = static_cast<float>(1.0 - a.beta2);
    c.eps = static_cast<float>(a.eps);
    c.decay = static_cast<float>(1.0 - a.lr * a.weight_decay);
    c.step_size = static_cast<float>(a.lr / (1.0 - pow(a.beta1, a.step)));
    c.inv_root = static_cast<float>(1.0 / sqrt(1.0 - pow(a.beta2, a.step)));
    c.step = a.step_dev;
    c.lr = a.lr_dev;
    c.lr_host = a.lr;
    c.wd = a.weight_decay;
    c.log_b1 = log(a.beta1);
    c.log_b2 = log(a.beta2);
    c.step_host = a.step;

    const uintptr_t wide = dtype == SLK_F32 ? 16 : 8, state = state_bits == 32 ? 16 : 4;
    for (int64_t i = 0; i < n_tensors; ++i) {
        const slk_adamw_tensor& t = tensors_host[i];
        if (t.n < 0) return fail(SLK_EINVAL, "adamw: negative size");
        if (t.n == 0) continue;
        if (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr ||
            t.exp_avg_sq == nullptr ||
            (state_bits == 8 && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr))) {
            return fail(SLK_EINVAL, "adamw: NULL pointer in tensor " + std::to_string(i));
        }
        if (ceil_div(t.n, kAdamSpan) > max_groups(kAdamThreads)) {
            return fail(SLK_EINVAL, "adamw: tensor " + std::to_string(i) + " is too large");
        }
    }
    AdamTable tab;
    tab.n = 0;
    tab.aligned = 0;
    int64_t groups = 0;
    auto launch = [&]() -> int {
        if (tab.n == 0) return SLK_OK;
        const dim3 grid(static_cast<unsigned>(groups)), wg(kAdamThreads);
        const hipStream_t st = as_stream(stream);
        if (dtype == SLK_F32) {
            if (state_bits == 8) hipLaunchKernelGGL((adamw_kernel<F32, true>), grid, wg, 0, st, tab, c);
            else hipLaunchKernelGGL((adamw_kernel<F32, false>), grid, wg, 0, st, tab, c);
        } else {
            if (state_bits == 8) hipLaunchKernelGGL((adamw_kernel<BF16, true>), grid, wg, 0, st, tab, c);
            else hipLaunchKernelGGL((adamw_kernel<BF16, false>), grid, wg, 0, st, tab, c);
        }
        tab.n = 0;
        tab.aligned = 0;
        groups = 0;
        return check_launch("adamw");
    };
    for (int64_t i = 0; i < n_tensors; ++i) {
        const slk_adamw_tensor& t = tensors_host[i];
        if (t.n == 0) continue;
        const int64_t need = ceil_div(t.n, kAdamSpan);
        if (tab.n == kAdamTensors || groups + need > max_groups(kAdamThreads)) {
            const int rc = launch();
            if (rc != SLK_OK) return rc;
        }
        tab.t[tab.n] = t;
        tab.first[tab.n] = static_cast<uint32_t>(groups);
        if (aligned_to(t.param, wide) && aligned_to(t.grad, wide) &&
            aligned_to(t.exp_avg, state) && aligned_to(t.exp_avg_sq, state)) {
            tab.aligned |= uint64_t{1} << tab.n;
        }
        ++tab.n;
        groups += need;
    }
    return launch();
}

extern "C" int slk_q8_decode(const void* codes, const float* scales, int64_t n, int is_signed,
                             float* out, void* stream) {
    using namespace slk;
    clear_error();
    if (n < 0) return fail(SLK_EINVAL, "q8_decode: negative size");
    if (n == 0) return SLK_OK;
    if (codes == nullptr || scales == nullptr || out == nullptr) {
        return fail(SLK_EINVAL, "q8_decode: NULL pointer");
    }
    const int64_t groups = ceil_div(n, kAdamSpan);
    if (groups > max_groups(kAdamThreads)) return fail(SLK_EINVAL, "q8_decode: too large");
    const bool al = aligned_to(codes, 4) && aligned_to(out, 16);
    const dim3 grid(static_cast<unsigned>(groups)), wg(kAdamThreads);
    if (is_signed) {
        hipLaunchKernelGGL((q8_decode_kernel<true>), grid, wg, 0, as_stream(stream), codes, scales,
                           n, al, out);
    } else {
        hipLaunchKernelGGL((q8_decode_kernel<false>), grid, wg, 0, as_stream(stream), codes,
                           scales, n, al, out);
    }
    return check_launch("q8_decode");
}

extern "C" int slk_q8_encode(const float* x, int64_t n, int is_signed, void* codes, float* scales,
                             void* stream) {
    using namespace slk;
    clear_error();
    if (n < 0) return fail(SLK_EINVAL, "q8_encode: negative size");
    if (n == 0) return SLK_OK;
    if (x == nullptr || scales == nullptr || codes == nullptr) {
        return fail(SLK_EINVAL, "q8_encode: NULL pointer");
    }
    const int64_t groups = ceil_div(n, kAdamSpan);
    if (groups > max_groups(kAdamThreads)) return fail(SLK_EINVAL, "q8_encode: too large");
    const bool al = aligned_to(codes, 4) && aligned_to(x, 16);
    const dim3 grid(static_cast<unsigned>(groups)), wg(kAdamThreads);
    if (is_signed) {
        hipLaunchKernelGGL((q8_encode_kernel<true>), grid, wg, 0, as_stream(stream), x, n, al,
                           codes, scales);
    } else {
        hipLaunchKernelGGL((q8_encode_kernel<false>), grid, wg, 0, as_stream(stream), x, n, al,
                           codes, scales);
    }
    return check_launch("q8_encode");
}

extern "C" int slk_carry_slots(const int32_t* row_start, int64_t nrows, int64_t total,
                               const int32_t* old_cols, const int32_t* old_nnz,
                               const int32_t* new_cols, const int32_t* new_nnz,
                               const slk_carry_state* states_host, int64_t n_states,
                               void* stream) {
    using namespace slk;
    clear_error();
    if (nrows < 0 || total < 0 || total > INT32_MAX || nrows > INT32_MAX) {
        return fail(SLK_EINVAL, "carry_slots: negative size, or slots beyond the int32 range");
    }
    if (n_states < 0 || n_states > SLK_CARRY_STATES || (n_states > 0 && states_host == nullptr)) {
        return fail(SLK_EINVAL, "carry_slots: between 0 and " + std::to_string(SLK_CARRY_STATES) +
                                    " states expected, got " + std::to_string(n_states));
    }
    if (total == 0 || n_states == 0) return SLK_OK;
    if (nrows == 0) return fail(SLK_EINVAL, "carry_slots: slots without rows");
    if (row_start == nullptr || old_cols == nullptr || old_nnz == nullptr ||
        new_cols == nullptr || new_nnz == nullptr) {
        return fail(SLK_EINVAL, "carry_slots: NULL structure array");
    }
    CarryTable tab;
    tab.n = static_cast<int32_t>(n_states);
    for (int64_t k = 0; k < n_states; ++k) {
        const slk_carry_state& s = states_host[k];
        if (s.kind != SLK_STATE_F32 && s.kind != SLK_STATE_Q8_SIGNED &&
            s.kind != SLK_STATE_Q8_UNSIGNED) {
            return fail(SLK_EINVAL, "carry_slots: unknown kind of state");
        }
        if (s.src == nullptr || s.dst == nullptr ||
            (s.kind != SLK_STATE_F32 && (s.src_scale == nullptr || s.dst_scale == nullptr))) {
            return fail(SLK_EINVAL, "carry_slots: NULL pointer in state " + std::to_string(k));
        }
        if (s.src == s.dst) {
            return fail(SLK_EINVAL, "carry_slots: a state cannot move in place");
        }
        tab.s[k] = s;
    }
    hipLaunchKernelGGL(carry_kernel, dim3(static_cast<unsigned>(ceil_div(total, kAdamSpan))),
                       dim3(kAdamThreads), 0, as_stream(stream), row_start, static_cast<int>(nrows),
                       static_cast<int>(total), old_cols,
                       old_nnz, new_cols, new_nnz, tab);
    return check_launch("carry_slots");
}
