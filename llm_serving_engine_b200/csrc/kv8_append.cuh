// RoPE + append to an 8-bit paged K/V cache: rotates q and k of the fused QKV output and
// quantises k and v into the cache's pages (the reference's write_kv_and_project_q,
// src/llm_serving_engine/model/model_runner.py:342-355, for a cache held in 8 bits).
//
//   cache   int8 [num_blocks, H_kv, block_size, D] (a page of one head is one contiguous run)
//           and one fp32 scale per (page, head), k and v each
//   page (b, h) with `old` tokens from earlier calls and this call's rows x:
//       s   = max(s_old if old > 0 else 0, max|x| / 127)
//       code of an earlier token:  rint(code * (s_old / s))   (only where s > s_old)
//       code of a new token:       clamp(rint(x / s), -127, 127)
//     a page of zeros has s = 0 and codes 0; a NaN or an infinity in x (or a NaN s_old) gives
//     s = NaN and codes 0, so that every value of the page reads back as NaN.
//   rotation of the first R of D dims:  out[d] = x[d] cos[d] + sign(d) x[partner(d)] sin[d],
//     half:        partner(d) = d + R/2 (sign -) for d < R/2, d - R/2 (sign +) above
//     interleaved: partner(d) = d + 1 (sign -) for even d, d - 1 (sign +) for odd d
//
// One warp per (page, KV head, k or v): it owns the page's scale, so no atomics.  Bound by
// latency for decode (one row per page) and by DRAM for prompts.
#pragma once

#include "common.cuh"

namespace lse {
namespace kv8 {

template <typename T>
struct AppendParams {
    const T *qkv;
    int64_t ld_qkv;
    const void *cos, *sin;
    int64_t ld_cs;
    int cs_type;  // 0 fp32, 1 bf16, 2 fp16
    int R, interleaved;
    T *q_out;  // [H, M, D]
    int8_t *pool[2];   // k, v
    float *scale[2];
    const int *block_table;
    int64_t bt_stride;
    int bt_cols;
    const int *query_offset, *q_start, *q_len;  // [E]
    int M, H, H_kv, D, E, num_blocks, block_size;
    int q_blocks;  // CTAs [0, q_blocks) rotate q, the rest append
};

constexpr int APPEND_THREADS = 256;

__device__ __forceinline__ float load_table(const void *p, int type, int64_t i) {
    if (type == 1) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    if (type == 2) return __half2float(static_cast<const __half *>(p)[i]);
    return static_cast<const float *>(p)[i];
}

// Element d of row m of a head whose elements start at `x`, rotated.
template <typename T>
__device__ __forceinline__ float rotated(const AppendParams<T> &p, const T *x, int m, int d) {
    const float a = to_float(x[d]);
    if (d >= p.R) return a;
    const int half = p.R / 2;
    const bool first = p.interleaved ? (d & 1) == 0 : d < half;
    const int pd = p.interleaved ? d ^ 1 : (first ? d + half : d - half);
    const float b = to_float(x[pd]);
    const int64_t c = m * p.ld_cs + d;
    const float cs = load_table(p.cos, p.cs_type, c), sn = load_table(p.sin, p.cs_type, c);
    return a * cs + (first ? -b : b) * sn;
}

template <typename T>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const AppendParams<T> p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");  // qkv is the previous kernel's output
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (static_cast<int>(blockIdx.x) < p.q_blocks) {
        const int64_t total = static_cast<int64_t>(p.M) * p.H * p.D;
        for (int64_t i = blockIdx.x * static_cast<int64_t>(APPEND_THREADS) + threadIdx.x; i < total;
             i += static_cast<int64_t>(p.q_blocks) * APPEND_THREADS) {
            const int d = static_cast<int>(i % p.D);
            const int64_t mh = i / p.D;
            const int h = static_cast<int>(mh % p.H), m = static_cast<int>(mh / p.H);
            const T *x = p.qkv + m * p.ld_qkv + static_cast<int64_t>(h) * p.D;
            p.q_out[(static_cast<int64_t>(h) * p.M + m) * p.D + d] = from_float<T>(rotated(p, x, m, d));
        }
        return;
    }
    __shared__ int s_pages[APPEND_THREADS];  // running sum of the pages that each entry touches
    const int warps = (gridDim.x - p.q_blocks) * (APPEND_THREADS / 32);
    const int me = (blockIdx.x - p.q_blocks) * (APPEND_THREADS / 32) + warp;
    for (int e0 = 0; e0 < p.E; e0 += APPEND_THREADS) {
        __syncthreads();
        {
            const int e = e0 + threadIdx.x;
            int n = 0;
            if (e < p.E) {
                const int len = p.q_len[e], off = p.query_offset[e];
                if (len > 0 && off >= 0) n = (off + len - 1) / p.block_size - off / p.block_size + 1;
            }
            s_pages[threadIdx.x] = n;
            __syncthreads();
            for (int k = 1; k < APPEND_THREADS; k <<= 1) {
                const int v = static_cast<int>(threadIdx.x) >= k ? s_pages[threadIdx.x - k] : 0;
                __syncthreads();
                s_pages[threadIdx.x] += v;
                __syncthreads();
            }
        }
        const int64_t items = static_cast<int64_t>(s_pages[APPEND_THREADS - 1]) * p.H_kv * 2;
        for (int64_t it = me; it < items; it += warps) {
            const int which = static_cast<int>(it & 1);
            const int h = static_cast<int>((it >> 1) % p.H_kv);
            const int pg = static_cast<int>((it >> 1) / p.H_kv);
            int lo = 0, hi = APPEND_THREADS - 1;  // the first entry whose running sum exceeds pg
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (s_pages[mid] > pg) hi = mid;
                else lo = mid + 1;
            }
            const int e = e0 + lo;
            const int off = p.query_offset[e], len = p.q_len[e], row0 = p.q_start[e];
            const int page = off / p.block_size + pg - (lo ? s_pages[lo - 1] : 0);
            const int first = max(off, page * p.block_size);
            const int last = min(off + len, (page + 1) * p.block_size);  // positions [first, last) are new
            const int old = first - page * p.block_size;
            const int blk = page < p.bt_cols ? p.block_table[e * p.bt_stride + page] : -1;
            if (blk < 0 || blk >= p.num_blocks || row0 < 0 || row0 + (last - off) > p.M) {
                if (lane == 0) report_status(LSE_ERR_INVALID_ARG);
                continue;
            }
            const T *x0 = p.qkv + static_cast<int64_t>(p.H + which * p.H_kv + h) * p.D;
            float top = 0.f;
            bool bad = false;
            for (int pos = first; pos < last; ++pos) {
                const int m = row0 + pos - off;
                const T *x = x0 + m * p.ld_qkv;
                for (int d = lane; d < p.D; d += 32) {
                    const float v = fabsf(which == 0 ? rotated(p, x, m, d) : to_float(x[d]));
                    bad |= !(v <= 3.402823466e38f);
                    top = fmaxf(top, v);
                }
            }
            for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            const int64_t cell = static_cast<int64_t>(blk) * p.H_kv + h;
            int8_t *dst = p.pool[which] + cell * p.block_size * p.D;
            const float s_old = old > 0 ? p.scale[which][cell] : 0.f;
            bad = __any_sync(0xffffffffu, bad || s_old != s_old);
            const float s = fmaxf(s_old, __fdiv_rn(top, 127.f));
            if (!bad && old > 0 && s > s_old) {  // the page's earlier tokens move to the larger scale
                const float f = __fdiv_rn(s_old, s);
                for (int i = lane; i < old * p.D; i += 32)
                    dst[i] = static_cast<int8_t>(rintf(static_cast<float>(dst[i]) * f));
            }
            for (int pos = first; pos < last; ++pos) {
                const int m = row0 + pos - off;
                const T *x = x0 + m * p.ld_qkv;
                int8_t *row = dst + (pos - page * p.block_size) * p.D;
                for (int d = lane; d < p.D; d += 32) {
                    const float v = which == 0 ? rotated(p, x, m, d) : to_float(x[d]);
                    float c = 0.f;
                    if (!bad && s > 0.f) c = fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.f), 127.f);
                    row[d] = static_cast<int8_t>(c);
                }
            }
            if (lane == 0) p.scale[which][cell] = bad ? __int_as_float(0x7fffffff) : s;
        }
    }
}

// Values of the pages ids[0..n): out[i, h, t, d] = code * scale, rounded once to T.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const int8_t *pool, const float *scale, int num_blocks, int H_kv,
                                                   int page_elems, const int64_t *ids, int64_t n, T *out) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t total = n * H_kv * page_elems;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x; i < total; i += gridDim.x * static_cast<int64_t>(256)) {
        const int64_t cell = i / page_elems;
        const int64_t b = ids[cell / H_kv];
        if (b < 0 || b >= num_blocks) {
            report_status(LSE_ERR_INVALID_ARG);
            out[i] = from_float<T>(0.f);
            continue;
        }
        const int64_t src = b * H_kv + cell % H_kv;
        out[i] = from_float<T>(static_cast<float>(pool[src * page_elems + i % page_elems]) * scale[src]);
    }
}

}  // namespace kv8
}  // namespace lse
