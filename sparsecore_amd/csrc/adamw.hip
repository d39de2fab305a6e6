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
// block of 8-bit codes, whose new scale is one wave reduction.
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
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int q = SIGNED ? q8_encode_signed(v[j], scale) : q8_encode_unsigned(v[j], scale);
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
        const float root = sqrtf(v[j]) * inv_root + c.eps;
        p[j] = p[j] * decay - step_size * (m[j] / root);
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

// One thread per four slots, one wave per SLK_Q8_BLOCK slots. Each live slot
// of the new topology looks its column up among its row's old columns (both
// ascending) and takes that slot's state; a grown connection and padding take
// 0. Out of place: a row's slots move both ways.
__global__ __launch_bounds__(kAdamThreads) void carry_kernel(
    const int32_t* __restrict__ row_start, int64_t nrows, int64_t total,
    const int32_t* __restrict__ old_cols, const int32_t* __restrict__ old_nnz,
    const int32_t* __restrict__ new_cols, const int32_t* __restrict__ new_nnz,
    const CarryTable tab) {
    const int64_t block = static_cast<int64_t>(blockIdx.x) * kAdamWaves + (threadIdx.x >> 6);
    const int lane = threadIdx.x & (kWave - 1);
    if (block * kQ8Block >= total) return;
    const int64_t i = block * kQ8Block + 4 * lane;

    // the row of slot i: the last that starts at or before it
    int64_t lo = 0, hi = nrows;  // row in [lo - 1, hi - 1]
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (row_start[mid] <= i) lo = mid + 1; else hi = mid;
    }
    int64_t row = lo - 1;
    int64_t from[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        from[j] = -1;
        const int64_t s = i + j;
        while (row + 1 < nrows && row_start[row + 1] <= s) ++row;
        if (s >= total || row < 0) continue;
        const int64_t start = row_start[row];
        if (s - start >= new_nnz[row]) continue;
        const int32_t col = new_cols[s];
        int64_t a = start, b = start + old_nnz[row];
        if (b > total) b = total;
        while (a < b) {
            const int64_t mid = (a + b) >> 1;
            if (old_cols[mid] < col) a = mid + 1; else b = mid;
        }
        const int64_t end = start + old_nnz[row];
        if (a < end && a < total && old_cols[a] == col) from[j] = a;
    }
    for (int k = 0; k < tab.n; ++k) {
        const slk_carry_state& st = tab.s[k];
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = 0.0f;
            if (from[j] < 0) continue;
            if (st.kind == SLK_STATE_F32) {
                v[j] = static_cast<const float*>(st.src)[from[j]];
            } else {
                const uint8_t q = static_cast<const uint8_t*>(st.src)[from[j]];
                const float scale = st.src_scale[from[j] / kQ8Block];
                v[j] = st.kind == SLK_STATE_Q8_SIGNED
                           ? q8_decode_signed(static_cast<int8_t>(q), scale)
                           : q8_decode_unsigned(q, scale);
            }
        }
        if (st.kind == SLK_STATE_F32) {
            const bool vec = i + 4 <= total && (reinterpret_cast<uintptr_t>(st.dst) & 15) == 0;
            store_some<F32>(st.dst, i, total, vec, v);
        } else {
            const bool vec = i + 4 <= total && (reinterpret_cast<uintptr_t>(st.dst) & 3) == 0;
            const float scale = q8_block_max(v);
            if (st.kind == SLK_STATE_Q8_SIGNED) encode4<true>(st.dst, i, total, vec, scale, v);
            else encode4<false>(st.dst, i, total, vec, scale, v);
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
        if (ceil_div(t.n, kAdamSpan) > INT32_MAX) {
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
        if (tab.n == kAdamTensors || groups + need > INT32_MAX) {
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
    if (groups > INT32_MAX) return fail(SLK_EINVAL, "q8_decode: too large");
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
    if (groups > INT32_MAX) return fail(SLK_EINVAL, "q8_encode: too large");
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
    if (nrows < 0 || total < 0 || total > INT32_MAX) {
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
                       dim3(kAdamThreads), 0, as_stream(stream), row_start, nrows, total, old_cols,
                       old_nnz, new_cols, new_nnz, tab);
    return check_launch("carry_slots");
}
