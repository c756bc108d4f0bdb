// Attention over the 8-bit paged K/V cache (kv8_append.cuh):
//
//   o[t, h, :] = softmax_p( scale * k_scale[b, g] * (q[t, h, :] . k_code[b, g, p % bs, :]) ) v_scale[b, g] v_code[b, g, p % bs, :]
//     b = block_table[e, p / bs], g = h / G, over the positions p < limit of the query.
//
// What its two kernels (kv8_decode.cuh, kv8_prompt.cuh) are given.
#pragma once

#include "common.cuh"

namespace lse {
namespace kv8 {

struct AttnParams {
    const void *q;  // element (t, h, d) at q[t * q_st + h * q_sh + d]
    int64_t q_st, q_sh;
    const int8_t *k_pool, *v_pool;  // [num_blocks, H_kv, block_size, D]
    const float *k_scale, *v_scale;  // [num_blocks, H_kv]
    const int *block_table;
    int64_t bt_stride;
    const int *context_len, *query_offset, *q_start, *q_len;  // query_offset null: one query per entry, at its end
    void *o;  // element (t, h, d) at o[t * o_st + h * o_sh + d]
    int64_t o_st, o_sh;
    int E, tokens, H, H_kv, bt_cols, block_size, num_blocks;
    float scale_log2;  // softmax scale * log2(e)
};

}  // namespace kv8
}  // namespace lse
