// Launcher of attention_decode.hip.
#pragma once

#include "attention.hpp"
#include "elem.hpp"

namespace slk {

struct AttnDecode {
    AttnArgs g;
    AttnIo q, k, v;
    const int32_t* k_lengths;  // live keys of each entry; NULL: all
    int32_t chunks;  // of a key head's rows
    int32_t vec;     // rows of K and V in 16-byte pieces
};

int attn_launch_decode(const AttnDecode& a, int db, int rows, hipStream_t st);

}  // namespace slk
