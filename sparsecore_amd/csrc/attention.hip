// slk_attention_*: argument checks, memory layout and launches.
#include <algorithm>

#include "attention.hpp"
#include "attention_decode.hpp"
#include "attention_prep.hpp"

namespace slk {

namespace {

constexpr int64_t kTileRows = kAttnTileRows;
// Rows of a key head (new tokens times the query heads of its group) that go the way
// of single tokens: it reads the keys once for four rows, the tiled way packs them
// once. 4 x 16384 keys, 32 heads over 8, bf16: 199 us against 257 with 16 rows, 349
// against 258 with 32; 16 x 2048 keys, 16 heads: 89 against 91 with 12, 101 with 16.
constexpr int64_t kFewRows = 16;
constexpr int64_t kCus = 256;

int64_t pad64(int64_t n) { return ceil_div(n, kAttnRows) * kAttnRows; }

bool packed_rows(const slk_attention& a) { return a.q_offsets != nullptr; }
bool uniform(const slk_attention& a) {
    return a.q_offsets == nullptr && a.q_lengths == nullptr && a.k_lengths == nullptr;
}

int blocks_of(int64_t dim) { return dim <= 32 ? 1 : dim <= 64 ? 2 : 4; }

struct Sizes {
    int64_t pad_q, pad_k;         // padded rows, an upper bound
    int64_t q_entries, k_entries; // tiles, an upper bound
    int64_t row;                  // bytes of a packed row
};

Sizes sizes_of(const slk_attention& a) {
    Sizes s;
    if (packed_rows(a)) {
        s.pad_q = pad64(a.rows_q) + kAttnRows * a.n;
        s.pad_k = pad64(a.rows_k) + kAttnRows * a.n;
        s.q_entries = a.rows_q / kTileRows + a.n + 2;
        s.k_entries = a.rows_k / kTileRows + a.n + 2;
    } else {
        s.pad_q = a.n * pad64(a.rows_q);
        s.pad_k = a.n * pad64(a.rows_k);
        s.q_entries = a.n * ceil_div(a.rows_q, kTileRows);
        s.k_entries = a.n * ceil_div(a.rows_k, kTileRows);
    }
    s.row = (a.dtype == SLK_F32 ? 4 : 2) * 32 * blocks_of(a.dim);
    return s;
}

// Consecutive pieces of a buffer, each 256-byte aligned.
struct Carver {
    char* base;
    int64_t at = 0;
    void* take(int64_t bytes) {
        void* p = base != nullptr ? base + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return p;
    }
};

struct Packed {
    char* data;
    int32_t* exps;
    uint64_t* bad;
    int8_t* rows;
};

Packed take_packed(Carver& c, const Sizes& s, int64_t heads, int64_t rows) {
    Packed p;
    p.data = static_cast<char*>(c.take(heads * rows * s.row));
    p.exps = static_cast<int32_t*>(c.take(heads * (rows / kAttnRows) * 4));
    p.bad = static_cast<uint64_t*>(c.take(heads * (rows / kAttnRows) * 8));
    p.rows = static_cast<int8_t*>(c.take(heads * rows));
    return p;
}

struct Plan {
    AttnSeq* seqs;
    int2 *q_list, *k_list;
    int32_t *count, *q_map, *k_map;
};

Plan take_plan(Carver& c, const slk_attention& a, const Sizes& s) {
    Plan p{};
    if (uniform(a)) return p;
    p.count = static_cast<int32_t*>(c.take(16));
    p.seqs = static_cast<AttnSeq*>(c.take((a.n + 2) * sizeof(AttnSeq)));
    p.q_map = static_cast<int32_t*>(c.take(s.pad_q / kAttnRows * 4));
    p.k_map = static_cast<int32_t*>(c.take(s.pad_k / kAttnRows * 4));
    p.q_list = static_cast<int2*>(c.take(s.q_entries * sizeof(int2)));
    if (a.keep) p.k_list = static_cast<int2*>(c.take(s.k_entries * sizeof(int2)));
    return p;
}

struct Saved {
    Plan plan;
    float *lse, *inv, *bias_rows;
    char* o_rest;
    Packed q, k, v;
    int64_t bytes;
};

Saved saved_of(const slk_attention& a, void* base) {
    const Sizes s = sizes_of(a);
    Carver c{static_cast<char*>(base)};
    Saved r{};
    r.plan = take_plan(c, a, s);
    r.lse = static_cast<float*>(c.take(a.heads * s.pad_q * 4));
    if (a.bias != nullptr) {
        r.inv = static_cast<float*>(c.take(a.heads * s.pad_q * 4));
        r.bias_rows = static_cast<float*>(c.take(a.heads * (2 * a.max_distance + 1) * 4));
    }
    if (a.dtype == SLK_BF16)
        r.o_rest = static_cast<char*>(c.take(a.heads * s.pad_q * 64 * blocks_of(a.dim)));
    r.q = take_packed(c, s, a.heads, s.pad_q);
    r.k = take_packed(c, s, a.kv_heads, s.pad_k);
    r.v = take_packed(c, s, a.kv_heads, s.pad_k);
    r.bytes = c.at;
    return r;
}

bool few_rows(const slk_attention& a) {
    return !a.keep && a.q_offsets == nullptr && a.q_lengths == nullptr &&
           a.heads / a.kv_heads * a.rows_q <= kFewRows;
}

struct Few {
    int rows, chunks, splits;
};

// Rows of a key head that a workgroup takes, and parts of the keys, at least 512
// each: as many workgroups as the card holds at once (by registers three a CU with
// one row, else two). 16 x 8192 keys, 32 heads over 8, 128 wide, bf16: 108 us with
// 512 workgroups, 120 with 1024, 168 with 256; 131071 keys, 12 heads, 64 wide,
// float32: 159 us with 768, 170 with 1032, 183 with 516.
Few few_of(const slk_attention& a) {
    const int64_t rows = a.heads / a.kv_heads * a.rows_q;
    Few f;
    f.rows = rows == 1 ? 1 : rows == 2 ? 2 : 4;
    f.chunks = static_cast<int>(ceil_div(rows, f.rows));
    const int64_t groups = a.n * a.kv_heads * f.chunks;
    const int64_t want = groups > 0 ? (f.rows == 1 ? 3 : 2) * kCus / groups : 1;
    const int64_t most = ceil_div(a.rows_k, 512);
    f.splits = static_cast<int>(
        std::max<int64_t>(1, std::min({want, most, int64_t{kAttnMaxSplits}})));
    return f;
}

// Parts of the keys in the tiled forward, where the query tiles leave CUs idle: two rounds
// of workgroups, parts of 256 keys or more. 128 x 8192 keys, 8 heads of 128, bfloat16: 45 us,
// unsplit 182; 1001 causal tokens, 12 heads of 64, float32: 37, unsplit 43, one round 40, parts
// of 128 keys 34 (but 54 for the first), of 512 keys 43; 512 tokens, 8 heads of 64, bfloat16:
// 23, unsplit 21, the join's price.
int splits_of(const slk_attention& a, const Sizes& s) {
    if (a.keep) return 1;
    const int64_t groups = s.q_entries * a.heads;
    if (groups == 0 || groups >= kCus) return 1;
    const int64_t most = a.rows_k / 256;
    return static_cast<int>(std::max<int64_t>(1, std::min({2 * kCus / groups, most, int64_t{kAttnMaxSplits}})));
}

struct Forward {
    Saved saved;  // its place, or a part of scratch
    float *part, *part_ml;
    int64_t part_rows;
    int splits;
    Few few;
    int64_t bytes;
};

Forward forward_of(const slk_attention& a, void* scratch) {
    const Sizes s = sizes_of(a);
    Carver c{static_cast<char*>(scratch)};
    Forward f{};
    if (few_rows(a)) {
        f.few = few_of(a);
        f.splits = f.few.splits;
    } else {
        f.splits = splits_of(a, s);
        if (a.keep) {
            f.saved = saved_of(a, a.saved);
        } else {
            f.saved = saved_of(a, c.base != nullptr ? c.base + c.at : nullptr);
            c.take(f.saved.bytes);
            f.saved.lse = nullptr;
        }
    }
    if (f.splits > 1) {
        // padded rows of queries; few queries are not padded
        f.part_rows = few_rows(a) ? a.n * a.rows_q : s.pad_q;
        const int64_t rows = f.splits * a.heads * f.part_rows;
        f.part = static_cast<float*>(c.take(rows * 32 * blocks_of(a.dim) * 4));
        f.part_ml = static_cast<float*>(c.take(rows * 8));
    }
    f.bytes = c.at;
    return f;
}

// Parts of a group's query heads in the keys' gradients: where the keys' tiles
// leave CUs idle, the heads go to workgroups of their own, whose sums are joined.
// Backward without dq, bfloat16, parts until there are four workgroups a CU: 8191 causal
// tokens, 16 heads over 4 of 128: 1113 us, 2098 in one part, 1355 with two a CU, 1102 with
// eight; 8 x 1024, 16 over 4 of 64: 139, 193, 145, 140; float32, 4 x 512, 16 over 2 of 64:
// 80, 264, 81, 80. The join of 8191 packed tokens' parts, 4 heads of 128: 25 us.
int dkv_parts(const slk_attention& a, const Sizes& s) {
    const int64_t rep = a.heads / a.kv_heads, groups = s.k_entries * a.kv_heads;
    int64_t parts = 1;
    while (parts < rep && groups * parts < 4 * kCus) {
        do ++parts;
        while (rep % parts != 0);
    }
    return static_cast<int>(parts);
}

struct Backward {
    int parts;
    float* dkv_part;
    float *delta, *lse;
    int32_t* dexps;
    int32_t* uneven;
    Packed dout;
    float* dbias_part;
    int64_t bytes;
};

Backward backward_of(const slk_attention& a, void* scratch) {
    const Sizes s = sizes_of(a);
    Carver c{static_cast<char*>(scratch)};
    Backward b{};
    b.delta = static_cast<float*>(c.take(a.heads * s.pad_q * 4));
    b.lse = static_cast<float*>(c.take(a.heads * s.pad_q * 4));
    b.dexps = static_cast<int32_t*>(c.take(a.heads * (s.pad_q / kAttnRows) * 4));
    b.uneven = static_cast<int32_t*>(c.take(4));
    b.dout = take_packed(c, s, a.heads, s.pad_q);
    b.parts = dkv_parts(a, s);
    if (b.parts > 1)
        b.dkv_part = static_cast<float*>(
            c.take(int64_t{b.parts} * 2 * a.kv_heads * s.pad_k * 32 * blocks_of(a.dim) * 4));
    if (a.dbias != nullptr)
        b.dbias_part = static_cast<float*>(
            c.take(a.heads * (s.pad_q / kAttnRows) * (2 * a.max_distance + 1) * 4));
    b.bytes = c.at;
    return b;
}

AttnIo io_of(const slk_attn_tensor& t) {
    return AttnIo{static_cast<char*>(t.p), t.batch, t.row, t.head, t.feature};
}

AttnOp op_of(const Packed& p, const Sizes& s, int64_t rows) {
    return AttnOp{p.data, rows * s.row, p.exps, p.bad, p.rows, rows / kAttnRows};
}

// Whether four elements that are consecutive along `unit` start at multiples of
// four of them: those of the other strides, and the pointer.
bool fours(const slk_attn_tensor& t, int64_t unit, int64_t a, int64_t b, int64_t c, int dtype) {
    return unit == 1 && a % 4 == 0 && b % 4 == 0 && c % 4 == 0 &&
           aligned_to(t.p, dtype == SLK_F32 ? 16 : 8);
}
bool four_features(const slk_attn_tensor& t, const slk_attention& a) {
    return a.dim % 4 == 0 && fours(t, t.feature, t.row, t.head, t.batch, a.dtype);
}

AttnVec vec_of(const slk_attn_tensor& t, const slk_attention& a) {
    const bool eight = a.dtype == SLK_BF16 && t.feature == 1 && aligned_to(t.p, 16) &&
                       (a.dim | t.row | t.head | t.batch) % 8 == 0;
    return eight                                                         ? kVecEight
           : four_features(t, a)                                         ? kVecFeatures
           : fours(t, t.row, t.feature, t.head, t.batch, a.dtype)        ? kVecRows
                                                                         : kVecNone;
}

AttnPackOp pack_op(const slk_attn_tensor& t, const Packed& p, const Sizes& s,
                   const slk_attention& a, bool keys, int64_t heads) {
    const int64_t rows = keys ? s.pad_k : s.pad_q;
    AttnPackOp o{};
    o.src = io_of(t);
    o.dst = p.data;
    o.dst_sh = rows * s.row;
    o.exps = p.exps;
    o.bad = p.bad;
    o.row_exps = p.rows;
    o.exps_sh = rows / kAttnRows;
    o.rows = rows;
    o.heads = static_cast<int32_t>(heads);
    o.keys = keys;
    o.vec = vec_of(t, a);
    return o;
}

AttnPlan plan_of(const slk_attention& a, const Plan& p, bool keys) {
    AttnPlan r{};
    r.seqs = p.seqs;
    r.list = keys ? p.k_list : p.q_list;
    r.count = p.count != nullptr ? p.count + (keys ? 2 : 0) : nullptr;
    r.q_map = p.q_map;
    r.k_map = p.k_map;
    r.batch = a.n;
    r.t = a.rows_q;
    r.s = a.rows_k;
    r.pad_t = pad64(a.rows_q);
    r.pad_s = pad64(a.rows_k);
    return r;
}

int make_plan(const slk_attention& a, const Plan& p, hipStream_t st) {
    if (p.seqs == nullptr) return SLK_OK;
    AttnPlanArgs g{};
    g.q_offsets = a.q_offsets;
    g.k_offsets = a.k_offsets != nullptr ? a.k_offsets : a.q_offsets;
    g.q_lengths = a.q_lengths;
    g.k_lengths = a.k_lengths;
    g.n = a.n;
    g.rows_q = a.rows_q;
    g.rows_k = a.rows_k;
    g.seqs = p.seqs;
    g.q_list = p.q_list;
    g.k_list = p.k_list;
    g.count = p.count;
    const Sizes s = sizes_of(a);
    g.q_map = p.q_map;
    g.k_map = p.k_map;
    g.q_tiles = s.pad_q / kAttnRows;
    g.k_tiles = s.pad_k / kAttnRows;
    g.causal = a.causal;
    while ((std::max(a.rows_q, a.rows_k) / kAttnRows) >> g.work_shift >= 1024) ++g.work_shift;
    return attn_launch_plan(g, st);
}

AttnArgs args_of(const slk_attention& a, float* bias_rows) {
    AttnArgs g{};
    g.vec_out = four_features(a.out, a);
    g.vec_q = four_features(a.dq, a);
    g.vec_kv = four_features(a.dk, a) && four_features(a.dv, a);
    g.out = io_of(a.out);
    g.dq = io_of(a.dq);
    g.dk = io_of(a.dk);
    g.dv = io_of(a.dv);
    g.lse_sh = sizes_of(a).pad_q;
    g.heads = static_cast<int32_t>(a.heads);
    g.kv_heads = static_cast<int32_t>(a.kv_heads);
    g.dim = static_cast<int32_t>(a.dim);
    g.dtype = a.dtype;
    g.causal = a.causal;
    g.splits = 1;
    g.scale = static_cast<float>(a.scale);
    g.scale2 = static_cast<float>(a.scale * 1.4426950408889634);
    if (a.bias != nullptr) {
        g.bias.table = a.bias;
        g.bias.rows = bias_rows;
        g.bias.dtype = a.bias_dtype;
        g.bias.buckets = static_cast<int32_t>(a.buckets);
        g.bias.max_distance = static_cast<int32_t>(a.max_distance);
        g.bias.one_sided = a.causal;
        const int64_t one = a.causal ? a.buckets : a.buckets / 2;
        for (int64_t i = 0; i < one; ++i)
            g.bias.starts[i] = static_cast<uint16_t>(a.bucket_starts[i]);
    }
    return g;
}

// Heads of queries, keys and values are one grid's second dimension.
bool heads_fit(const slk_attention& a) {
    return a.heads >= 1 && a.kv_heads >= 1 && a.heads % a.kv_heads == 0 && a.heads <= 16384;
}

// Padded rows of all heads are counted in 64 bits, rows in 32. Rows and sequences are
// bounded before they are multiplied.
bool rows_fit(const slk_attention& a) {
    if (a.n > INT32_MAX / 64 || a.rows_q > INT32_MAX / 2 || a.rows_k > INT32_MAX / 2) return false;
    const Sizes s = sizes_of(a);
    return s.pad_q <= INT32_MAX / 2 && s.pad_k <= INT32_MAX / 2;
}

// Whether memory can be counted for these arguments; check() says what is wrong with others.
bool countable(const slk_attention* a) {
    return a != nullptr && a->n >= 0 && a->rows_q >= 0 && a->rows_k >= 0 && a->dim >= 1 &&
           a->dim <= SLK_ATTN_MAX_DIM && heads_fit(*a) && rows_fit(*a) &&
           (a->bias == nullptr ||
            (a->max_distance >= 1 && a->max_distance <= SLK_ATTN_MAX_DISTANCE));
}

int check(const slk_attention* args, const char* who, bool backward) {
    const std::string w = who;
    if (args == nullptr) return fail(SLK_EINVAL, w + ": NULL arguments");
    const slk_attention& a = *args;
    if (a.n < 0 || a.rows_q < 0 || a.rows_k < 0) return fail(SLK_EINVAL, w + ": negative size");
    if (a.dtype != SLK_F32 && a.dtype != SLK_BF16)
        return fail(SLK_EINVAL, w + ": unknown dtype " + std::to_string(a.dtype));
    if (a.dim < 1 || a.dim > SLK_ATTN_MAX_DIM)
        return fail(SLK_EINVAL, w + ": dim in [1, " + std::to_string(SLK_ATTN_MAX_DIM) +
                                    "], got " + std::to_string(a.dim));
    if (!heads_fit(a))
        return fail(SLK_EINVAL, w + ": heads must be a multiple of kv_heads, at most 16384, got " +
                                    std::to_string(a.heads) + " and " +
                                    std::to_string(a.kv_heads));
    // times log2 e it is a float32
    if (!(a.scale >= 0.0) || !(a.scale <= 2e38))
        return fail(SLK_EINVAL, w + ": scale must be finite and not negative, at most 2e38");
    if (packed_rows(a) && (a.q_lengths != nullptr || a.k_lengths != nullptr))
        return fail(SLK_EINVAL, w + ": offsets or lengths, not both");
    if (!packed_rows(a) && a.k_offsets != nullptr)
        return fail(SLK_EINVAL, w + ": k_offsets need q_offsets");
    if (packed_rows(a) && a.k_offsets == nullptr && a.rows_q != a.rows_k)
        return fail(SLK_EINVAL, w + ": queries and keys share offsets but not their rows");
    if (a.bias != nullptr) {
        if (a.bias_dtype != SLK_F32 && a.bias_dtype != SLK_BF16)
            return fail(SLK_EINVAL, w + ": unknown bias dtype");
        const int64_t one = a.causal ? a.buckets : a.buckets / 2;
        if (a.buckets < 1 || a.buckets > SLK_ATTN_MAX_BUCKETS || one < 1 ||
            (!a.causal && a.buckets % 2 != 0))
            return fail(SLK_EINVAL, w + ": buckets in [1, " +
                                        std::to_string(SLK_ATTN_MAX_BUCKETS) +
                                        "], even where both sides are seen");
        if (a.max_distance < 1 || a.max_distance > SLK_ATTN_MAX_DISTANCE)
            return fail(SLK_EINVAL, w + ": max_distance in [1, " +
                                        std::to_string(SLK_ATTN_MAX_DISTANCE) + "]");
        if (a.bucket_starts == nullptr || a.bucket_starts[0] != 0)
            return fail(SLK_EINVAL, w + ": bucket_starts must begin with 0");
        for (int64_t i = 1; i < one; ++i)
            if (a.bucket_starts[i] < a.bucket_starts[i - 1] ||
                a.bucket_starts[i] > a.max_distance)
                return fail(SLK_EINVAL, w + ": bucket_starts must ascend to max_distance at most");
    }
    if (a.n == 0 && !packed_rows(a)) return SLK_OK;
    if (!rows_fit(a)) return fail(SLK_EINVAL, w + ": too many rows");
    const Sizes s = sizes_of(a);
    if (s.q_entries * a.heads > max_groups(kAttnThreads) ||
        s.k_entries * a.heads > max_groups(kAttnThreads) || s.pad_q > max_groups(kWave) ||
        s.pad_k > max_groups(kAttnThreads) * 32)
        return fail(SLK_EINVAL, w + ": too many tiles");
    if (!backward) {
        if (a.rows_q > 0 && (a.q.p == nullptr || a.out.p == nullptr))
            return fail(SLK_EINVAL, w + ": NULL q or out");
        if (a.rows_k > 0 && (a.k.p == nullptr || a.v.p == nullptr))
            return fail(SLK_EINVAL, w + ": NULL k or v");
    } else {
        if (a.rows_q > 0 && (a.out.p == nullptr || a.dout.p == nullptr))
            return fail(SLK_EINVAL, w + ": NULL out or dout");
        if ((a.dk.p == nullptr) != (a.dv.p == nullptr))
            return fail(SLK_EINVAL, w + ": dk and dv go together");
        if (a.dbias != nullptr && a.bias == nullptr)
            return fail(SLK_EINVAL, w + ": dbias without a bias");
    }
    if (a.keep || backward) {
        const int64_t need = saved_of(a, nullptr).bytes;
        if (need > 0 && (a.saved == nullptr || a.saved_bytes < need))
            return fail(SLK_EINVAL, w + ": saved too small (need " + std::to_string(need) + ")");
    }
    const int64_t need = backward ? backward_of(a, nullptr).bytes : forward_of(a, nullptr).bytes;
    if (need > 0 && (a.scratch == nullptr || a.scratch_bytes < need))
        return fail(SLK_EINVAL, w + ": scratch too small (need " + std::to_string(need) + ")");
    if (!aligned_to(a.saved, 16) || !aligned_to(a.scratch, 16))
        return fail(SLK_EINVAL, w + ": saved and scratch must be 16-byte aligned");
    return SLK_OK;
}

int few_forward(const slk_attention& a, const Forward& f, hipStream_t st) {
    AttnDecode d{};
    d.g = args_of(a, nullptr);
    d.g.plan = plan_of(a, f.saved.plan, false);
    d.g.splits = f.splits;
    d.g.part = f.part;
    d.g.part_ml = f.part_ml;
    d.g.part_rows = f.part_rows;
    d.g.plan.pad_t = a.rows_q;
    d.q = io_of(a.q);
    d.k = io_of(a.k);
    d.v = io_of(a.v);
    d.k_lengths = a.k_lengths;
    d.chunks = f.few.chunks;
    const int64_t unit = a.dtype == SLK_F32 ? 4 : 8;
    auto pieces = [&](const slk_attn_tensor& t) {
        return t.feature == 1 && a.dim % 8 == 0 && t.row % unit == 0 && t.head % unit == 0 &&
               t.batch % unit == 0 && aligned_to(t.p, 16);
    };
    d.vec = pieces(a.k) && pieces(a.v);
    return attn_launch_decode(d, blocks_of(a.dim), f.few.rows, st);
}

}  // namespace

}  // namespace slk

extern "C" int64_t slk_attention_saved_bytes(const slk_attention* args) {
    return slk::countable(args) && args->keep ? slk::saved_of(*args, nullptr).bytes : 0;
}

extern "C" int64_t slk_attention_scratch_bytes(const slk_attention* args, int backward) {
    if (!slk::countable(args)) return 0;
    return backward ? slk::backward_of(*args, nullptr).bytes
                    : slk::forward_of(*args, nullptr).bytes;
}

extern "C" int slk_attention_forward(const slk_attention* args, void* stream) {
    using namespace slk;
    clear_error();
    int rc = check(args, "attention_forward", false);
    if (rc != SLK_OK) return rc;
    const slk_attention& a = *args;
    if (a.n == 0 && !packed_rows(a)) return SLK_OK;
    const hipStream_t st = as_stream(stream);
    // without queries too the backward has keys' gradients to write, by the plan's list
    if (a.rows_q == 0) return a.keep ? make_plan(a, saved_of(a, a.saved).plan, st) : SLK_OK;
    const Forward f = forward_of(a, a.scratch);
    if (few_rows(a)) return few_forward(a, f, st);
    const Sizes s = sizes_of(a);
    const bool split = a.dtype == SLK_F32;
    rc = make_plan(a, f.saved.plan, st);
    if (rc != SLK_OK) return rc;

    AttnArgs g = args_of(a, f.saved.bias_rows);
    g.plan = plan_of(a, f.saved.plan, false);
    AttnPack p{};
    p.plan = g.plan;
    p.dim = g.dim;
    p.heads = g.heads;
    p.bias = g.bias;
    p.n = 3;
    p.op[0] = pack_op(a.q, f.saved.q, s, a, false, a.heads);
    p.op[1] = pack_op(a.k, f.saved.k, s, a, true, a.kv_heads);
    p.op[2] = pack_op(a.v, f.saved.v, s, a, true, a.kv_heads);
    rc = attn_launch_pack(p, blocks_of(a.dim), a.dtype, st);
    if (rc != SLK_OK) return rc;
    g.tiles = ceil_div(a.rows_q, kTileRows);
    g.q = op_of(f.saved.q, s, s.pad_q);
    g.k = op_of(f.saved.k, s, s.pad_k);
    g.v = op_of(f.saved.v, s, s.pad_k);
    g.lse = f.saved.lse;
    g.inv = f.saved.inv;
    g.o_rest = a.keep ? f.saved.o_rest : nullptr;
    g.splits = f.splits;
    g.part = f.part;
    g.part_ml = f.part_ml;
    g.part_rows = f.part_rows;
    return attn_launch_forward(g, split, blocks_of(a.dim), s.q_entries, st);
}

extern "C" int slk_attention_backward(const slk_attention* args, void* stream) {
    using namespace slk;
    clear_error();
    int rc = check(args, "attention_backward", true);
    if (rc != SLK_OK) return rc;
    const slk_attention& a = *args;
    const hipStream_t st = as_stream(stream);
    if (a.n == 0 && !packed_rows(a)) {  // nothing to sum: zeros
        return a.dbias != nullptr ? attn_launch_dbias(args_of(a, nullptr), a.dbias, st) : SLK_OK;
    }
    const Sizes s = sizes_of(a);
    const bool split = a.dtype == SLK_F32;
    const Saved sv = saved_of(a, a.saved);
    const Backward b = backward_of(a, a.scratch);
    AttnArgs g = args_of(a, sv.bias_rows);
    g.plan = plan_of(a, sv.plan, false);
    if (a.rows_q > 0) {
        AttnPack p{};
        p.plan = g.plan;
        p.dim = g.dim;
        p.n = 1;
        p.op[0] = pack_op(a.dout, b.dout, s, a, false, a.heads);
        p.o = io_of(a.out);
        p.o_vec = vec_of(a.out, a);
        p.o_rest = sv.o_rest;
        p.delta = b.delta;
        p.delta_sh = s.pad_q;
        p.lse = sv.lse;
        p.lse_out = b.lse;
        p.dexps = b.dexps;
        p.clear = b.uneven;
        rc = attn_launch_pack(p, blocks_of(a.dim), a.dtype, st);
        if (rc != SLK_OK) return rc;
    }
    g.tiles = ceil_div(a.rows_q, kTileRows);
    g.q = op_of(sv.q, s, s.pad_q);
    g.k = op_of(sv.k, s, s.pad_k);
    g.v = op_of(sv.v, s, s.pad_k);
    g.dout = op_of(b.dout, s, s.pad_q);
    g.lse = b.lse;
    g.inv = sv.inv;
    g.delta = b.delta;
    g.dexps = b.dexps;
    g.uneven = b.uneven;
    g.dbias_part = b.dbias_part;
    g.dkv_part = b.dkv_part;
    g.dkv_rows = s.pad_k;
    g.dkv_parts = b.parts;
    g.dbias_slots = s.pad_q / kAttnRows;
    const bool want_q = a.rows_q > 0 && (a.dq.p != nullptr || a.dbias != nullptr);
    const bool want_kv = a.rows_k > 0 && a.dk.p != nullptr;
    rc = attn_launch_backward(g, split, blocks_of(a.dim), plan_of(a, sv.plan, true), s.q_entries,
                              s.k_entries, want_q, want_kv, ceil_div(a.rows_k, kTileRows), st);
    if (rc != SLK_OK || a.dbias == nullptr) return rc;
    return attn_launch_dbias(g, a.dbias, st);
}
