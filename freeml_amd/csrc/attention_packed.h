// Arguments of the packed attention kernels (attention_packed.hip).
#pragma once

#include "fmlh_internal.h"

namespace fmlh {

struct PackedAttn {
    uint32_t n_seq, q_rows, k_rows;
    int group;     // query heads per key head
    uint32_t n_kv; // key heads
    int head_dim;
    float scale;
    int vec;       // every row and head 16-byte aligned, head_dim a multiple of 4
    const int32_t *q_off, *k_off, *k_len;
    size_t q_rs, k_rs, v_rs, o_rs, k_hs, v_hs;
};

}  // namespace fmlh
