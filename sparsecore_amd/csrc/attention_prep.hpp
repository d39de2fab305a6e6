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
    int32_t* count;  // tiles of queries, their padded rows, tiles of keys, padded rows
    int32_t tile_q, tile_k, causal, work_shift;
};

struct AttnPackOp {
    AttnIo src;
    char* dst;       // NULL: delta only
    int64_t dst_sr, dst_sh;
    int32_t* exps;
    int64_t exps_sh, rows;
    int32_t heads, keys;
};

struct AttnPack {
    AttnPlan plan;
    AttnPackOp op[3];
    int32_t n, dim;
    AttnIo o;        // with delta: op[0] is dO, this is O
    float* delta;
    int64_t delta_sh;
    int32_t* dexps;
};

int attn_launch_plan(const AttnPlanArgs& a, hipStream_t st);
int attn_launch_pack(const AttnPack& a, bool split, int db, int dtype, hipStream_t st);

}  // namespace slk
