// Log-probabilities of given tokens, entropy and top alternatives of rows of logits:
//
//   Z = sum_v exp(x[v] - max x),  logprob = x[token] - max x - log Z
//   entropy = log Z - sum_v (x[v] - max x) exp(x[v] - max x) / Z
//   top: the k largest x (equal ones by index, lowest first) and their log-probabilities
//
// A row without any x above -inf has log-probabilities -inf and entropy 0; a row holding a
// NaN or +inf has NaN for both.  In the order of the alternatives a NaN comes first.
#pragma once

#include "common.cuh"

namespace lse {
namespace logprobs {

struct Params {
    const void *x;  // [M, V], row stride ld
    int64_t ld;
    const int64_t *tokens;  // [M] or null
    float *logprob, *entropy;  // [M]; logprob null without tokens
    float *top_logprob;     // [M, k]
    int64_t *top_id;        // [M, k]
    int M, V, k;
};

constexpr int THREADS = 256;

__device__ __forceinline__ float to_float(float v) { return v; }
using lse::to_float;

// Order of the alternatives as an unsigned integer: larger value first, NaN above all.
__device__ __forceinline__ unsigned order_of(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __float_as_uint(x + 0.f);  // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Params p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float s_a[THREADS], s_b[THREADS];
    __shared__ unsigned long long s_key[THREADS];
    const T *x = static_cast<const T *>(p.x) + blockIdx.x * p.ld;
    float top = -INFINITY;
    bool nan = false;
    for (int v = threadIdx.x; v < p.V; v += THREADS) {
        const float a = to_float(x[v]);
        nan |= a != a || a == INFINITY;
        top = fmaxf(top, a);
    }
    nan = __syncthreads_or(nan);
    s_a[threadIdx.x] = top;
    for (int k = THREADS / 2; k > 0; k >>= 1) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < k) s_a[threadIdx.x] = fmaxf(s_a[threadIdx.x], s_a[threadIdx.x + k]);
    }
    __syncthreads();
    top = s_a[0];
    __syncthreads();
    float z = 0.f, w = 0.f;
    for (int v = threadIdx.x; v < p.V; v += THREADS) {
        const float d = to_float(x[v]) - top, e = d == -INFINITY || top == -INFINITY ? 0.f : expf(d);
        z += e;
        if (e > 0.f) w = fmaf(d, e, w);
    }
    s_a[threadIdx.x] = z;
    s_b[threadIdx.x] = w;
    for (int k = THREADS / 2; k > 0; k >>= 1) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < k) {
            s_a[threadIdx.x] += s_a[threadIdx.x + k];
            s_b[threadIdx.x] += s_b[threadIdx.x + k];
        }
    }
    __syncthreads();
    z = s_a[0];
    w = s_b[0];
    const bool empty = top == -INFINITY && !nan;
    const float log_z = logf(z), none = __int_as_float(0x7fffffff);
    auto lp = [&](float a) { return nan ? none : empty ? -INFINITY : (a - top) - log_z; };
    if (threadIdx.x == 0) {
        p.entropy[blockIdx.x] = nan ? none : empty ? 0.f : log_z - w / z;
        if (p.tokens) {
            const int64_t t = p.tokens[blockIdx.x];
            const bool in = t >= 0 && t < p.V;
            if (!in) report_status(LSE_ERR_INVALID_ARG);
            p.logprob[blockIdx.x] = in ? lp(to_float(x[t])) : none;
        }
    }
    unsigned long long last = ~0ull;
    for (int r = 0; r < p.k; ++r) {
        unsigned long long best = 0;
        for (int v = threadIdx.x; v < p.V; v += THREADS) {
            const unsigned long long key = (static_cast<unsigned long long>(order_of(to_float(x[v]))) << 32) | (0x7fffffffu - v);
            if (key < last && key > best) best = key;
        }
        s_key[threadIdx.x] = best;
        for (int k = THREADS / 2; k > 0; k >>= 1) {
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < k && s_key[threadIdx.x + k] > s_key[threadIdx.x]) s_key[threadIdx.x] = s_key[threadIdx.x + k];
        }
        __syncthreads();
        last = s_key[0];
        __syncthreads();
        if (threadIdx.x == 0) {
            const int64_t at = blockIdx.x * static_cast<int64_t>(p.k) + r;
            p.top_id[at] = 0x7fffffffu - static_cast<unsigned>(last);
            p.top_logprob[at] = lp(value_of(static_cast<unsigned>(last >> 32)));
        }
    }
}

}  // namespace logprobs
}  // namespace lse
