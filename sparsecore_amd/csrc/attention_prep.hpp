// Launchers of attention_prep.hip.
#pragma once

#include "attention.hpp"

namespace slk {

struct AttnPlanArgs {
    const int32_t *q_offsets, *k_offsets;  // packed rows: n + 1 each; or NULL and
    const int32_t *q_lengths, *k_lengths;  // live rows of batch entries (NULL: all)
    int64_t n, rows_q, rows_k;             // rows of the arrays, or of a batch entry
    AttnSeq* seqs;                         // n (+ 2 if packed)
    int2 *q_list, *k_list;                 // NULL: not wanted
    int32_t *q_map, *k_map;                // sequences of q_tiles and k_tiles tiles of 64
    int64_t q_tiles, k_tiles;
    int32_t* count;  // tiles of queries, their padded rows, tiles of keys, padded rows
    int32_t causal, work_shift;
};

// What a pack reads at once: an element, four features, four rows, eight features.
enum AttnVec { kVecNone = 0, kVecFeatures = 1, kVecRows = 2, kVecEight = 3 };

struct AttnPackOp {
    AttnIo src;
    char* dst;
    int64_t dst_sh;
    int32_t* exps;
    uint64_t* bad;
    int8_t* row_exps;
    int64_t exps_sh, rows;
    int32_t heads, keys, vec;
};

struct AttnPack {
    AttnPlan plan;
    AttnPackOp op[3];
    int32_t n, dim, heads;
    AttnBias bias;   // with a table: its rows are made too
    AttnIo o;        // with delta: op[0] is dO, this is O
    int32_t o_vec;
    char* o_rest;    // what rounding took off O (bfloat16)
    float* delta;
    const float* lse;
    float* lse_out;  // lse, NaN where a row of dO is not finite
    int64_t delta_sh;
    int32_t* dexps;
    int32_t* clear;  // with delta: set to 0
};

int attn_launch_plan(const AttnPlanArgs& a, hipStream_t st);
int attn_launch_pack(const AttnPack& a, int db, int dtype, hipStream_t st);

}  // namespace slk
