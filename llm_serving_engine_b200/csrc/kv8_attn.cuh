// Attention over the 8-bit paged K/V cache (kv8_append.cuh):
//
//   o[t, h, :] = softmax_p( scale * k_scale[b, g] * (q[t, h, :] . k_code[b, g, p % bs, :]) ) v_scale[b, g] v_code[b, g, p % bs, :]
//     b = block_table[e, p / bs], g = h / G, over the positions p < limit of the query.
//
// One warp per (query, head): a position at a time, fp32 throughout.
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

template <int D, typename T>
__global__ void __launch_bounds__(256) attn_rows_kernel(const AttnParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int W = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t rows = static_cast<int64_t>(p.tokens) * p.H;
    if (blockIdx.x == 0 && p.query_offset != nullptr)  // rows outside q are never reached: say so
        for (int e = threadIdx.x; e < p.E; e += 256)
            if (p.q_len[e] > 0 && (p.q_start[e] < 0 || p.q_start[e] > p.tokens - p.q_len[e])) report_status(LSE_ERR_INVALID_ARG);
    for (int64_t r = blockIdx.x * 8ll + warp; r < rows; r += gridDim.x * 8ll) {
        const int t = static_cast<int>(r / p.H), h = static_cast<int>(r % p.H);
        int e = -1, limit = 0;
        if (p.query_offset == nullptr) {
            e = t;
            limit = p.context_len[e];
        } else {
            for (int e0 = 0; e0 < p.E && e < 0; e0 += 32) {
                const int c = e0 + lane;
                const bool in = c < p.E && t >= p.q_start[c] && t - p.q_start[c] < p.q_len[c];
                const unsigned hit = __ballot_sync(0xffffffffu, in);
                if (hit) e = e0 + __ffs(hit) - 1;
            }
            if (e < 0) continue;  // a row of no entry is not written
            limit = min(p.context_len[e], p.query_offset[e] + t - p.q_start[e] + 1);
        }
        if (limit > p.bt_cols * static_cast<int64_t>(p.block_size)) {
            if (lane == 0) report_status(LSE_ERR_INVALID_ARG);
            limit = p.bt_cols * p.block_size;
        }
        const int g = h / (p.H / p.H_kv);
        const T *q = static_cast<const T *>(p.q) + t * p.q_st + h * p.q_sh;
        float qv[W], acc[W], m = -INFINITY, l = 0.f;
        for (int i = 0; i < W; ++i) {
            qv[i] = to_float(q[lane * W + i]);
            acc[i] = 0.f;
        }
        for (int pos = 0; pos < limit; ++pos) {
            const int blk = p.block_table[e * p.bt_stride + pos / p.block_size];
            if (blk < 0 || blk >= p.num_blocks) {
                if (lane == 0) report_status(LSE_ERR_INVALID_ARG);
                continue;
            }
            const int64_t cell = static_cast<int64_t>(blk) * p.H_kv + g;
            const int64_t at = (cell * p.block_size + pos % p.block_size) * D + lane * W;
            float s = 0.f;
            for (int i = 0; i < W; ++i) s = fmaf(qv[i], static_cast<float>(p.k_pool[at + i]), s);
            for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
            s *= p.scale_log2 * p.k_scale[cell];
            const float mn = s != s ? s : fmaxf(m, s);  // a NaN score stays
            const float f = m == mn ? 1.f : exp2f(m - mn), w = exp2f(s - mn);
            m = mn;
            l = l * f + w;
            const float wv = w * p.v_scale[cell];
            for (int i = 0; i < W; ++i) acc[i] = acc[i] * f + wv * static_cast<float>(p.v_pool[at + i]);
        }
        T *o = static_cast<T *>(p.o) + t * p.o_st + h * p.o_sh;
        for (int i = 0; i < W; ++i) o[lane * W + i] = from_float<T>(limit > 0 && l != 0.f ? acc[i] / l : 0.f);
    }
}

}  // namespace kv8
}  // namespace lse
