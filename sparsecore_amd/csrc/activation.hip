// An activation between two layers, y = f(x), and what its backward needs of x in
// 8 bits (slk_activation_*).
//
// Codes. SLK_ACT_BLOCK consecutive elements share a float32 scale, the largest
// finite magnitude `top` of them; x is kept as q = round(x · (127 / top)), the
// value q · (top · (1/127)): off by at most top / 254. Each operation is one
// correctly rounded float32 operation in the order written, so codes do not
// depend on the kernel that makes them. top < 2^-100 keeps zeros; an element that
// is not finite has the code -128 and is NaN again, its neighbours keep theirs,
// and the block's scale is stored with its sign bit set, so that the others need
// not look for such codes.
//
// One pass each way: x in, y and the codes out; dy and the codes in, dx out. What
// bounds it is memory. A wave takes whole blocks, four elements a lane, four
// blocks at a time where there are enough of them (loads of all four in flight).
// 8191 x 16384 bfloat16, SiLU: forward and backward 260 us, 5.2 TB/s.
#include "elem.hpp"

namespace slk {

namespace {

constexpr int kActBlock = SLK_ACT_BLOCK;
static_assert(kActBlock == 4 * kWave, "four elements a lane: a wave holds one block");
constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kManyBlocks = 4;  // blocks a wave takes at a time, of large arrays

// 0.5·erfc(|x| / sqrt 2) and exp(-x^2 / 2), for results that are rounded to
// bfloat16. Their ratio as a polynomial in t = 1 / (1 + 0.36 |x|), fitted for the
// smallest relative error on [0, 14]: 2^-20.1, so the tail keeps its digits, where a
// polynomial for erfc itself is good to 1e-7 absolutely (off by 0.4% of f at -6, by
// 3% at -12). The exponential's argument, rounded, adds 2^-19 up to |x| = 3 and 2^-17
// at 13. (erfcf takes some 60 instructions, and with it the kernel was bound by them.)
__device__ __forceinline__ float half_erfc_fast(float x, float& bell) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, fabsf(x), 1.0f));
    bell = __builtin_amdgcn_exp2f(-0.72134752f * x * x);
    float p = __builtin_fmaf(t, 0.04700576f, -0.17958629f);
    p = __builtin_fmaf(t, p, 0.18070686f);
    p = __builtin_fmaf(t, p, 0.02671937f);
    p = __builtin_fmaf(t, p, 0.13965873f);
    p = __builtin_fmaf(t, p, 0.14178291f);
    p = __builtin_fmaf(t, p, 0.14371236f);
    return t * p * bell;
}

// 1 / (1 + exp(-x))
template <bool FAST>
__device__ __forceinline__ float logistic(float x) {
    if constexpr (FAST)
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * x));
    else return 1.0f / (1.0f + expf(-x));
}

// f and its derivative. Float32, relative errors of a few 2^-24 of |f| + |x f'|;
// FAST, for results that are rounded to bfloat16: 2^-19 of them up to |x| = 3, 2^-16
// down to where they leave the normal numbers (an exponential's argument of up to 126
// carries 2^-24 of itself).
template <int KIND, bool FAST>
__device__ __forceinline__ float act(float x) {
    if constexpr (KIND == SLK_ACT_RELU) {
        return x <= 0.0f ? 0.0f : x;
    } else if constexpr (KIND == SLK_ACT_SILU) {
        if constexpr (FAST) return x * logistic<true>(x);
        else return x / (1.0f + expf(-x));
    } else if constexpr (KIND == SLK_ACT_GELU) {
        if constexpr (FAST) {
            float bell;
            const float h = half_erfc_fast(x, bell);
            return x * (x < 0.0f ? h : 1.0f - h);
        }
        // x·Phi(x) by the complement, which keeps its digits for negative x
        return 0.5f * x * erfcf(-0.70710678f * x);
    } else if constexpr (KIND == SLK_ACT_GELU_TANH) {
        // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3)
        const float u2 = 1.5957691f * __builtin_fmaf(0.044715f * x * x, x, x);
        if constexpr (FAST) return x * logistic<true>(u2);
        else return x / (1.0f + expf(-u2));
    } else {
        return x;
    }
}

template <int KIND, bool FAST>
__device__ __forceinline__ float slope(float x) {
    if constexpr (KIND == SLK_ACT_RELU) {
        return x > 0.0f ? 1.0f : x <= 0.0f ? 0.0f : x;
    } else if constexpr (KIND == SLK_ACT_SILU) {
        const float s = logistic<FAST>(x);
        return s * __builtin_fmaf(x, 1.0f - s, 1.0f);
    } else if constexpr (KIND == SLK_ACT_GELU) {
        if constexpr (FAST) {
            float bell;
            const float h = half_erfc_fast(x, bell);
            return __builtin_fmaf(x * 0.39894228f, bell, x < 0.0f ? h : 1.0f - h);
        }
        return __builtin_fmaf(x * 0.39894228f, expf(-0.5f * x * x), 0.5f * erfcf(-0.70710678f * x));
    } else if constexpr (KIND == SLK_ACT_GELU_TANH) {
        const float u2 = 1.5957691f * __builtin_fmaf(0.044715f * x * x, x, x);
        const float d2 = 1.5957691f * __builtin_fmaf(0.134145f * x, x, 1.0f);
        const float s = logistic<FAST>(u2);
        // s (1 - s) is 0 where u2 overflows; x d2 is not to make NaN of it
        const float t = s * (1.0f - s);
        return t == 0.0f ? s : __builtin_fmaf(x * d2, t, s);
    } else {
        return 1.0f;
    }
}

template <class IO>
__device__ __forceinline__ void load_four(const void* p, int64_t i, int64_t n, bool vec,
                                          float (&v)[4]) {
    if (vec && i + 4 <= n) {
        IO::load4(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j < n ? IO::load(p, i + j) : 0.0f;
    }
}

template <class IO>
__device__ __forceinline__ void store_four(void* p, int64_t i, int64_t n, bool vec,
                                           const float (&v)[4]) {
    if (vec && i + 4 <= n) {
        IO::store4(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) IO::store(p, i + j, v[j]);
    }
}

// Maximum over the wave's lanes, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t m) {
    auto dpp = [&](auto ctrl) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
            0, static_cast<int>(m), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    m = max(m, dpp(std::integral_constant<int, 0xb1>{}));   // lanes 1, 0, 3, 2 of four
    m = max(m, dpp(std::integral_constant<int, 0x4e>{}));   // lanes 2, 3, 0, 1
    m = max(m, dpp(std::integral_constant<int, 0x141>{}));  // half-row mirror
    m = max(m, dpp(std::integral_constant<int, 0x140>{}));  // row mirror
    m = max(m, static_cast<uint32_t>(__shfl_xor(m, 16)));
    return max(m, static_cast<uint32_t>(__shfl_xor(m, 32)));
}

// Codes of a block's four elements of a lane, in one word; its scale in every
// lane. x + 1.5·2^23 rounds to the nearest whole number (ties to even) and holds
// it in its low bits.
__device__ __forceinline__ uint32_t encode(const float (&x)[4], float& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    m = __builtin_amdgcn_readfirstlane(wave_max(m));
    const bool odd = m >= 0x7f800000u;  // the same for all lanes
    if (odd) {
        m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t b = __float_as_uint(x[j]) & 0x7fffffffu;
            if (b < 0x7f800000u) m = max(m, b);
        }
        m = __builtin_amdgcn_readfirstlane(wave_max(m));
    }
    const float top = __uint_as_float(m);
    const float inv = top >= 0x1p-100f ? 127.0f / top : 0.0f;
    scale = __uint_as_float(m | (odd ? 0x80000000u : 0u));
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float r = x[j] * inv + 12582912.0f;
        w |= (__float_as_uint(r) & 0xffu) << (8 * j);
    }
    if (odd) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((__float_as_uint(x[j]) & 0x7fffffffu) >= 0x7f800000u)
                w = (w & ~(0xffu << (8 * j))) | (0x80u << (8 * j));
    }
    return w;
}

__device__ __forceinline__ void decode(uint32_t w, float scale, float (&x)[4]) {
    const float top = fabsf(scale);
    const float step = top >= 0x1p-100f ? top * (1.0f / 127.0f) : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        x[j] = static_cast<float>(static_cast<int>(w << (24 - 8 * j)) >> 24) * step;
    if (__float_as_uint(scale) >> 31) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (((w >> (8 * j)) & 0xffu) == 0x80u) x[j] = __builtin_nanf("");
    }
}

__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int64_t i, int64_t n, bool vec) {
    if (vec && i + 4 <= n) return *reinterpret_cast<const uint32_t*>(p + i);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) w |= static_cast<uint32_t>(p[i + j]) << (8 * j);
    return w;
}

__device__ __forceinline__ void store_codes(uint8_t* p, int64_t i, int64_t n, bool vec,
                                            uint32_t w) {
    if (vec && i + 4 <= n) {
        *reinterpret_cast<uint32_t*>(p + i) = w;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) p[i + j] = static_cast<uint8_t>(w >> (8 * j));
}

struct ActArgs {
    const void* x;
    void* y;
    const void* dy;
    void* dx;
    uint8_t* codes;
    float* scales;
    int64_t n;
    bool vec_x, vec_y, vec_codes;  // x or dy; y or dx; codes: aligned for four at once
};

__device__ __forceinline__ int64_t first_block(int per) {
    const int64_t wave = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    return wave * per;
}

template <class IO, int KIND, int PER>
__global__ __launch_bounds__(kThreads) void act_forward_kernel(const ActArgs a) {
    const int64_t b0 = first_block(PER);
    float x[PER][4];
#pragma unroll
    for (int b = 0; b < PER; ++b)
        load_four<IO>(a.x, (b0 + b) * kActBlock + 4 * (threadIdx.x & 63), a.n, a.vec_x, x[b]);
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        const int64_t at = (b0 + b) * kActBlock + 4 * (threadIdx.x & 63);
        if ((b0 + b) * kActBlock >= a.n) return;  // the same for all lanes
        if (a.codes != nullptr) {
            float scale;
            const uint32_t w = encode(x[b], scale);
            store_codes(a.codes, at, a.n, a.vec_codes, w);
            if ((threadIdx.x & 63) == 0) a.scales[b0 + b] = scale;
        }
        if (a.y != nullptr) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = act<KIND, IO::kBytes == 2>(x[b][j]);
            store_four<IO>(a.y, at, a.n, a.vec_y, y);
        }
    }
}

// dx = dy · f'(x) with x from its codes, or from x itself where there are none.
// dy NULL: dx is x.
template <class IO, int KIND, int PER>
__global__ __launch_bounds__(kThreads) void act_backward_kernel(const ActArgs a) {
    const int64_t b0 = first_block(PER);
    float dy[PER][4], x[PER][4];
    uint32_t w[PER];
    float scale[PER];
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        const int64_t at = (b0 + b) * kActBlock + 4 * (threadIdx.x & 63);
        if (a.codes != nullptr) {
            w[b] = load_codes(a.codes, at, a.n, a.vec_codes);
            scale[b] = (b0 + b) * kActBlock < a.n ? a.scales[b0 + b] : 0.0f;
        } else {
            load_four<IO>(a.x, at, a.n, a.vec_codes, x[b]);
        }
        if (a.dy != nullptr) load_four<IO>(a.dy, at, a.n, a.vec_x, dy[b]);
    }
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        const int64_t at = (b0 + b) * kActBlock + 4 * (threadIdx.x & 63);
        if ((b0 + b) * kActBlock >= a.n) return;
        if (a.codes != nullptr) decode(w[b], scale[b], x[b]);
        float dx[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            dx[j] = a.dy != nullptr ? dy[b][j] * slope<KIND, IO::kBytes == 2>(x[b][j]) : x[b][j];
        store_four<IO>(a.dx, at, a.n, a.vec_y, dx);
    }
}

template <class IO, int KIND, int PER>
void launch(const ActArgs& a, bool backward, hipStream_t st) {
    const int64_t groups = ceil_div(ceil_div(a.n, kActBlock), PER * kWaves);
    const dim3 grid(static_cast<unsigned>(groups)), wg(kThreads);
    if (backward) hipLaunchKernelGGL((act_backward_kernel<IO, KIND, PER>), grid, wg, 0, st, a);
    else hipLaunchKernelGGL((act_forward_kernel<IO, KIND, PER>), grid, wg, 0, st, a);
}

template <class IO, int KIND>
void launch_per(const ActArgs& a, bool backward, hipStream_t st) {
    // four blocks a wave once that still fills the card four times over
    if (a.n >= int64_t{kActBlock} * kManyBlocks * kWaves * 1024)
        launch<IO, KIND, kManyBlocks>(a, backward, st);
    else launch<IO, KIND, 1>(a, backward, st);
}

template <class IO>
void launch_kind(const ActArgs& a, int kind, bool backward, hipStream_t st) {
    switch (kind) {
        case SLK_ACT_RELU: return launch_per<IO, SLK_ACT_RELU>(a, backward, st);
        case SLK_ACT_SILU: return launch_per<IO, SLK_ACT_SILU>(a, backward, st);
        case SLK_ACT_GELU: return launch_per<IO, SLK_ACT_GELU>(a, backward, st);
        case SLK_ACT_GELU_TANH: return launch_per<IO, SLK_ACT_GELU_TANH>(a, backward, st);
        default: return launch_per<IO, SLK_ACT_NONE>(a, backward, st);
    }
}

int run(const slk_activation* args, bool backward, const char* who, void* stream) {
    clear_error();
    const std::string w = who;
    if (args == nullptr) return fail(SLK_EINVAL, w + ": NULL arguments");
    const slk_activation& g = *args;
    if (g.n < 0) return fail(SLK_EINVAL, w + ": negative size");
    if (g.dtype != SLK_F32 && g.dtype != SLK_BF16)
        return fail(SLK_EINVAL, w + ": unknown dtype " + std::to_string(g.dtype));
    if (g.kind < SLK_ACT_NONE || g.kind > SLK_ACT_GELU_TANH)
        return fail(SLK_EINVAL, w + ": unknown kind " + std::to_string(g.kind));
    if (ceil_div(g.n, kActBlock) > max_groups(kThreads))
        return fail(SLK_EINVAL, w + ": too large");
    if (g.n == 0) return SLK_OK;
    if ((g.codes == nullptr) != (g.scales == nullptr))
        return fail(SLK_EINVAL, w + ": codes and scales go together");
    if (backward ? g.dx == nullptr || (g.codes == nullptr && g.x == nullptr)
                 : g.x == nullptr || (g.y == nullptr && g.codes == nullptr))
        return fail(SLK_EINVAL, w + ": NULL pointer");
    const uintptr_t four = g.dtype == SLK_F32 ? 16 : 8;
    ActArgs a{};
    a.x = g.x;
    a.y = g.y;
    a.dy = g.dy;
    a.dx = g.dx;
    a.codes = g.codes;
    a.scales = g.scales;
    a.n = g.n;
    a.vec_x = aligned_to(backward ? g.dy : g.x, four);
    a.vec_y = aligned_to(backward ? g.dx : g.y, four);
    a.vec_codes = g.codes != nullptr ? aligned_to(g.codes, 4) : aligned_to(g.x, four);
    const hipStream_t st = as_stream(stream);
    if (g.dtype == SLK_F32) launch_kind<F32>(a, g.kind, backward, st);
    else launch_kind<BF16>(a, g.kind, backward, st);
    return check_launch(who);
}

}  // namespace

}  // namespace slk

extern "C" int slk_activation_forward(const slk_activation* args, void* stream) {
    return slk::run(args, false, "activation_forward", stream);
}

extern "C" int slk_activation_backward(const slk_activation* args, void* stream) {
    return slk::run(args, true, "activation_backward", stream);
}
