// Arguments of the packed attention kernels (attention_packed.hip).
#pragma once

#include "fmlh_internal.h"

namespace fmlh {

// Row stride in floats up to which a tile of 64 rows lies inside the 31 bits of a buffer's offsets.
constexpr size_t kMaxVecStride = size_t(1) << 22;

struct PackedAttn {
    uint32_t n_seq, q_rows, k_rows;
    int group;     // query heads per key head
    uint32_t n_kv; // key heads
    int head_dim;
    float scale;
    int vec;       // every row and head 16-byte aligned, head_dim a multiple of 4, row strides up to kMaxVecStride
    const int32_t *q_off, *k_off, *k_len;
    size_t q_rs, k_rs, v_rs, o_rs, k_hs, v_hs;
};

// The kernels on the bf16 matrix cores (attention_packed_split.hip).  Grids hold `items` / `tiles` per
// key head; ws, delta and sums are workspace.
int attn_split_forward(const PackedAttn& a, int per, uint32_t items, uint32_t budget, float* out, float* lse, const float* q,
                       const float* k, const float* v, float* ws, hipStream_t s);
// Rows, or keys, of a tile of the backward pass.
int attn_split_dq_rows(const PackedAttn& a);
int attn_split_back_rows(const PackedAttn& a);
// Floats that one of the parts of dk and dv leaves in `sums` (parts > 1).
size_t attn_split_part_floats(const PackedAttn& a, uint32_t key_tiles);
int attn_split_backward(const PackedAttn& a, uint32_t row_tiles, uint32_t key_tiles, int parts, float* dq, float* dk, float* dv,
                        float* delta, const float* dout, const float* out, const float* lse, const float* q, const float* k,
                        const float* v, float* sums, hipStream_t s);

}  // namespace fmlh
