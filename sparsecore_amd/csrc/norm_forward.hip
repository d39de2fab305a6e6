// Forward of the residual norm, slk_norm_forward:
//   r = x + scale · gate ∘ post(branch),   y = pre(r)
// One pass: a token's features stay in registers from the first load to the
// last store, so each array moves once (16 bytes a feature in float32) and the
// kernel is bound by memory. 16384 x 4096 bfloat16 with both norms and a gate takes
// 158 us under the profiler; with its backward 308 to 317 us outside it, 4.2 to 4.4
// TB/s. 8192 x 384 float32 feature-major 12.9 us, eight tokens 2.9.
#include "norm.hpp"

namespace slk {
namespace {

struct FwdRow {
    const void *x, *gate, *weight, *bias, *post_weight, *post_bias;
    float* stats;
    int64_t n, per_gate;  // tokens that share a row of gate
    int d;
    bool layer, has_branch;
    float scale, eps, inv_d;
};

// r and y of token n from its branch features u (changed in place: r) and x,
// which is in y.
template <class T, int EPL, int TW, bool VEC, class Sum>
__device__ __forceinline__ void forward_row(const FwdRow& p, int64_t n, int l, float (&u)[EPL],
                                            float (&y)[EPL], Sum& sum) {
    float s[EPL];
    float pmean = 0.0f, prstd = 0.0f;
    if (p.has_branch) {
        if (p.post_weight != nullptr) {
            row_stats<EPL, TW, VEC>(u, p.d, l, p.layer, p.inv_d, p.eps, sum, pmean, prstd);
            row_load<T, EPL, TW, VEC>(p.post_weight, 0, p.d, l, s);
#pragma unroll
            for (int q = 0; q < EPL; ++q) u[q] = (u[q] - pmean) * prstd * s[q];
            if (p.post_bias != nullptr) {
                row_load<T, EPL, TW, VEC>(p.post_bias, 0, p.d, l, s);
#pragma unroll
                for (int q = 0; q < EPL; ++q) u[q] += s[q];
            }
        }
        if (p.gate != nullptr) {
            row_load<T, EPL, TW, VEC>(p.gate, n / p.per_gate * p.d, p.d, l, s);
#pragma unroll
            for (int q = 0; q < EPL; ++q) u[q] *= s[q];
        }
#pragma unroll
        for (int q = 0; q < EPL; ++q) u[q] = y[q] + p.scale * u[q];
    } else {
#pragma unroll
        for (int q = 0; q < EPL; ++q) u[q] = y[q];
    }
    float mean, rstd;
    row_stats<EPL, TW, VEC>(u, p.d, l, p.layer, p.inv_d, p.eps, sum, mean, rstd);
    row_load<T, EPL, TW, VEC>(p.weight, 0, p.d, l, s);
#pragma unroll
    for (int q = 0; q < EPL; ++q) y[q] = (u[q] - mean) * rstd * s[q];
    if (p.bias != nullptr) {
        row_load<T, EPL, TW, VEC>(p.bias, 0, p.d, l, s);
#pragma unroll
        for (int q = 0; q < EPL; ++q) y[q] += s[q];
    }
    if (p.stats != nullptr && l == 0) {
        f32x4 st = {mean, rstd, pmean, prstd};
        *reinterpret_cast<f32x4*>(p.stats + 4 * n) = st;
    }
}

// All arrays token-major: a token a team.
template <class T, int EPL, int TW, bool VEC>
__global__ __launch_bounds__(TW > 4 ? TW * kWave : kNormThreads) void norm_forward_kernel(
    const FwdRow p, const void* __restrict__ branch, void* __restrict__ r, void* __restrict__ y) {
    __shared__ float red[2 * TW];
    TeamSum<TW, 1> sum{red};
    const int l = TW == 1 ? threadIdx.x & (kWave - 1) : threadIdx.x;
    const int64_t n = TW == 1 ? static_cast<int64_t>(blockIdx.x) * (kNormThreads / kWave) +
                                    __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                              : blockIdx.x;
    if (n >= p.n) return;  // a whole team
    float u[EPL], v[EPL];
    row_load<T, EPL, TW, VEC>(p.x, n * p.d, p.d, l, v);
    if (p.has_branch) row_load<T, EPL, TW, VEC>(branch, n * p.d, p.d, l, u);
    forward_row<T, EPL, TW, VEC>(p, n, l, u, v, sum);
    if (p.has_branch) row_store<T, EPL, TW, VEC>(r, n * p.d, p.d, l, u);
    row_store<T, EPL, TW, VEC>(y, n * p.d, p.d, l, v);
}

// branch or y feature-major: TT tokens a workgroup, the feature-major arrays
// through one LDS tile (y overwrites the branch token by token).
template <class T, int EPL, int TT, bool VEC>
__global__ __launch_bounds__(kTileThreads) void norm_forward_tile_kernel(
    const FwdRow p, const void* __restrict__ branch, void* __restrict__ r, void* __restrict__ y,
    int branch_cols, int y_cols, int pairs) {
    extern __shared__ float tile[];
    TeamSum<1, 1> sum{nullptr};
    const int l = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = xcd_logical_block(blockIdx.x, gridDim.x) * TT;
    Ahead<T, EPL, VEC, true> x;
    if (n0 + wv < p.n) x.fetch(p.x, (n0 + wv) * p.d, p.d, l);
    if (branch_cols) {
        tile_load<T, TT>(branch, p.n, p.d, n0, pairs, tile);
        __syncthreads();
    }
#pragma unroll 1  // unrolled, the tokens' registers add up
    for (int t = wv; t < TT; t += kTileWaves) {
        const int64_t n = n0 + t;
        if (n >= p.n) break;
        float u[EPL], v[EPL];
        x.get(p.x, n * p.d, p.d, l, v);
        if (t + kTileWaves < TT && n + kTileWaves < p.n)
            x.fetch(p.x, (n + kTileWaves) * p.d, p.d, l);
        if (p.has_branch) {
            if (branch_cols) tile_row_load<EPL, TT, VEC>(tile, t, p.d, l, u);
            else row_load<T, EPL, 1, VEC>(branch, n * p.d, p.d, l, u);
        }
        forward_row<T, EPL, 1, VEC>(p, n, l, u, v, sum);
        if (p.has_branch) row_store<T, EPL, 1, VEC>(r, n * p.d, p.d, l, u);
        if (y_cols) tile_row_store<EPL, TT, VEC>(tile, t, p.d, l, v);
        else row_store<T, EPL, 1, VEC>(y, n * p.d, p.d, l, v);
    }
    if (y_cols) {
        __syncthreads();
        tile_store<T, TT>(y, p.n, p.d, n0, pairs, tile);
    }
}

template <class T>
int forward(const slk_norm* a, const FwdRow& p, hipStream_t st) {
    const bool cols = (a->branch_cols && a->branch != nullptr) || a->y_cols;
    if (cols) {
        // two workgroups a CU: 65536 x 768 float32 takes 200 us at 16 tokens, 241 at 32
        const int tokens = tile_tokens(a->n, p.d, 75 * 1024);
        const int pairs = tile_pairs(a, {a->branch_cols ? a->branch : nullptr,
                                         a->y_cols ? a->y : nullptr});
        const bool vec = norm_vec(a, {a->x, a->branch_cols ? nullptr : a->branch, a->gate,
                                      a->weight, a->bias, a->post_weight, a->post_bias, a->r,
                                      a->y_cols ? nullptr : a->y});
        const dim3 grid(static_cast<unsigned>(ceil_div(a->n, tokens))), wg(kTileThreads);
        const size_t lds = 4 * static_cast<size_t>(tile_quarter(p.d)) * (tokens + 1) * sizeof(float);
        auto go = [&](auto kv, auto ks) {
            if (vec) {
                hipLaunchKernelGGL(kv, grid, wg, lds, st, p, a->branch, a->r, a->y,
                                   a->branch_cols, a->y_cols, pairs);
            } else {
                hipLaunchKernelGGL(ks, grid, wg, lds, st, p, a->branch, a->r, a->y,
                                   a->branch_cols, a->y_cols, pairs);
            }
        };
        auto pick = [&](auto epl, auto tt) {
            constexpr int E = decltype(epl)::value, TT = decltype(tt)::value;
            go(norm_forward_tile_kernel<T, E, TT, true>, norm_forward_tile_kernel<T, E, TT, false>);
        };
        using std::integral_constant;
        if (p.d <= 512 && tokens == 32) pick(integral_constant<int, 8>{}, integral_constant<int, 32>{});
        else if (p.d <= 512) pick(integral_constant<int, 8>{}, integral_constant<int, 16>{});
        else if (tokens == 32) pick(integral_constant<int, 16>{}, integral_constant<int, 32>{});
        else pick(integral_constant<int, 16>{}, integral_constant<int, 16>{});
        return check_launch("norm_forward");
    }
    const bool vec = norm_vec(a, {a->x, a->branch, a->gate, a->weight, a->bias, a->post_weight,
                                  a->post_bias, a->r, a->y});
    norm_shape(p.d, [&](auto epl, auto tw) {
        constexpr int E = decltype(epl)::value, W = decltype(tw)::value;
        const dim3 grid(static_cast<unsigned>(W == 1 ? ceil_div(a->n, kNormThreads / kWave) : a->n));
        const dim3 wg(W == 1 ? kNormThreads : W * kWave);
        if (vec) {
            hipLaunchKernelGGL((norm_forward_kernel<T, E, W, true>), grid, wg, 0, st, p, a->branch,
                               a->r, a->y);
        } else {
            hipLaunchKernelGGL((norm_forward_kernel<T, E, W, false>), grid, wg, 0, st, p,
                               a->branch, a->r, a->y);
        }
    });
    return check_launch("norm_forward");
}

}  // namespace

int validate_norm(const slk_norm* a, const char* who, bool backward) {
    const std::string w(who);
    if (a == nullptr) return fail(SLK_EINVAL, w + ": NULL arguments");
    if (a->n < 0 || a->d < 1 || a->d > SLK_NORM_MAX_D) {
        return fail(SLK_EINVAL, w + ": n must be >= 0 and d in [1, " +
                                    std::to_string(SLK_NORM_MAX_D) + "], got n=" +
                                    std::to_string(a->n) + ", d=" + std::to_string(a->d));
    }
    if (a->dtype != SLK_F32 && a->dtype != SLK_BF16) {
        return fail(SLK_EINVAL, w + ": dtype must be SLK_F32 or SLK_BF16");
    }
    // threads of a token: a tile has 16 tokens at least, a row kernel a team each
    int64_t threads = kTileThreads / 16;
    if (!a->branch_cols && !a->y_cols)
        norm_shape(static_cast<int>(a->d), [&](auto, auto tw) { threads = tw * kWave; });
    const int64_t most = max_groups(threads) - 64;  // (the last workgroup's may be idle)
    if (a->n > most) {
        return fail(SLK_EINVAL, w + ": at most " + std::to_string(most) + " tokens of d=" +
                                    std::to_string(a->d) + " in a call, got n=" +
                                    std::to_string(a->n));
    }
    if ((a->branch_cols || a->y_cols) && a->d > SLK_NORM_COLS_MAX) {
        return fail(SLK_EINVAL, w + ": feature-major arrays need d <= " +
                                    std::to_string(SLK_NORM_COLS_MAX));
    }
    if (a->gate != nullptr && a->branch == nullptr) {
        return fail(SLK_EINVAL, w + ": a gate needs a branch");
    }
    if (a->post_weight != nullptr && a->branch == nullptr) {
        return fail(SLK_EINVAL, w + ": a post norm needs a branch");
    }
    if (a->post_bias != nullptr && a->post_weight == nullptr) {
        return fail(SLK_EINVAL, w + ": post_bias needs post_weight");
    }
    if (!a->layer && (a->bias != nullptr || a->post_bias != nullptr)) {
        return fail(SLK_EINVAL, w + ": RMSNorm has no bias");
    }
    if (a->gate != nullptr && a->n > 0 && (a->gate_rows < 1 || a->n % a->gate_rows != 0)) {
        return fail(SLK_EINVAL, w + ": gate_rows=" + std::to_string(a->gate_rows) +
                                    " must divide n=" + std::to_string(a->n));
    }
    if (a->weight == nullptr) return fail(SLK_EINVAL, w + ": NULL weight");
    if (a->n > 0 && !backward && (a->x == nullptr || a->y == nullptr ||
                                  (a->branch != nullptr && a->r == nullptr))) {
        return fail(SLK_EINVAL, w + ": NULL x, r or y");
    }
    if (!aligned_to(a->stats, 16)) {
        return fail(SLK_EINVAL, w + ": stats must be 16-byte aligned");
    }
    if (a->n > 0 && backward && (a->r == nullptr || a->stats == nullptr)) {
        return fail(SLK_EINVAL, w + ": NULL r or stats");
    }
    return SLK_OK;
}

}  // namespace slk

extern "C" int slk_norm_forward(const slk_norm* a, void* stream) {
    using namespace slk;
    clear_error();
    const int rc = validate_norm(a, "norm_forward", false);
    if (rc != SLK_OK || a->n == 0) return rc;
    FwdRow p;
    p.x = a->x;
    p.gate = a->gate;
    p.weight = a->weight;
    p.bias = a->bias;
    p.post_weight = a->post_weight;
    p.post_bias = a->post_bias;
    p.stats = a->stats;
    p.n = a->n;
    p.per_gate = a->gate != nullptr ? a->n / a->gate_rows : 1;
    p.d = static_cast<int>(a->d);
    p.layer = a->layer != 0;
    p.has_branch = a->branch != nullptr;
    p.scale = static_cast<float>(a->scale);
    p.eps = static_cast<float>(a->eps);
    p.inv_d = 1.0f / static_cast<float>(a->d);
    return a->dtype == SLK_F32 ? forward<F32>(a, p, as_stream(stream))
                               : forward<BF16>(a, p, as_stream(stream));
}
