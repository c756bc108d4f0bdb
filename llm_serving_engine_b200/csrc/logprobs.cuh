// Log-probabilities of given tokens, entropy and top alternatives of rows of logits:
//
//   Z = sum_v exp(x[v] - max x),  logprob = x[token] - max x - log Z
//   entropy = log Z - sum_v (x[v] - max x) exp(x[v] - max x) / Z
//   top: the k largest x (equal ones by index, lowest first) and their log-probabilities
//
// A row without any x above -inf has log-probabilities -inf and entropy 0; a row holding a
// NaN or +inf has NaN for both.  In the order of the alternatives a NaN comes first.
//
// One pass over the row, bound by DRAM where there are many rows and by latency where there are
// few:
//   * a warp reads a group of GROUP consecutive logits with 16-byte loads, takes its maximum,
//     moves its running maximum m if it has to, and adds exp(x - m) and (x - m) exp(x - m) to its lanes'
//     fp32 sums; with few rows a cluster of up to 8 CTAs shares one, joined through
//     distributed shared memory;
//   * the alternatives come out of the groups' maxima: ordered by (maximum, index), the first k
//     groups hold the k largest logits (of k other groups, each has an element that comes before
//     any element of a group after them), so only those are read again, and of them only what
//     reaches the k-th group's maximum is ranked.  A short row has few groups; there every
//     lane's 16 bytes are a group of their own.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace lse {
namespace logprobs {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_GROUPS = 1024;   // groups of a CTA
constexpr int MAX_TOP = LSE_LOGPROBS_MAX_TOP;
constexpr int CANDIDATES = 512;    // logits ranked directly; more go round by round

struct Params {
    const void *x;  // [M, V], row stride ld
    int64_t ld;
    const int64_t *tokens;  // [M] or null
    float *logprob, *entropy;  // [M]; logprob null without tokens
    float *top_logprob;     // [M, k]
    int64_t *top_id;        // [M, k]
    int M, V, k;
    int cluster;  // CTAs of a row
    int group;    // logits of a group (a multiple of a warp's load of 32 x 16 bytes, x 2)
    int groups;   // groups of a CTA (rounded up)
    int fine;     // the alternatives come from the maxima of single 16-byte loads (short rows)
};

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
constexpr unsigned ORDER_INF = 0xff800000u, ORDER_NONE = 0x007fffffu;  // of +inf and -inf

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error 2^-22; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes of logits as floats.
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float operator[](int i) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = *reinterpret_cast<const __half2 *>(&w[i / 2]);
            return i & 1 ? __high2float(h) : __low2float(h);
        } else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    // The largest, a NaN if there is one.
    __device__ __forceinline__ float top() const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (std::is_same_v<T, float>) {
            float m = __uint_as_float(w[0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(w[i])));
            return m;
        } else {
            using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
            T2 m = *reinterpret_cast<const T2 *>(&w[0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, *reinterpret_cast<const T2 *>(&w[i]));
            return lse::to_float(__hmax_nan(m.x, m.y));
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Params p) {
    constexpr int N = Vec<T>::N, STEP = 64 * N;  // logits of a warp's two loads
    __shared__ unsigned s_top[MAX_GROUPS];       // order of each group's maximum
    __shared__ unsigned s_all[MAX_CLUSTER * 256];  // the row's (rank 0; fewer groups a CTA when it shares a row)
    __shared__ float s_sum[WARPS][3];            // m, sum of exp, sum of (x - m) exp
    __shared__ float s_row[3];                   // this CTA's
    __shared__ int s_count, s_sel_n, s_sel[MAX_TOP];
    __shared__ unsigned long long s_key[CANDIDATES];
    __shared__ unsigned long long s_best[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const T *x = static_cast<const T *>(p.x) + row * p.ld;
    // Elements are numbered from the 16-byte boundary at or before the row, so that loads are aligned;
    // `shift` of them belong to what is before it and are not touched.
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    const T *x0 = x - shift;
    const int64_t end = static_cast<int64_t>(p.V) + shift;
    const int64_t cta0 = static_cast<int64_t>(rank) * p.groups * p.group;  // this CTA's first element
    auto load = [&](int64_t at) {
        Vec<T> v;
        if (at >= shift && at + N <= end) {
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v.raw.x), "=r"(v.raw.y), "=r"(v.raw.z), "=r"(v.raw.w) : "l"(x0 + at));
        } else {  // an end of the row: -inf in the place of what is outside
            T e[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = at + i >= shift && at + i < end;
                if constexpr (std::is_same_v<T, float>) e[i] = in ? x0[at + i] : -INFINITY;
                else e[i] = in ? x0[at + i] : from_float<T>(-INFINITY);
            }
            v.raw = *reinterpret_cast<const uint4 *>(e);
        }
        return v;
    };

    // ---- the pass: warp w takes groups w, w + WARPS, ... of this CTA -----------------------------------
    float m = -INFINITY, z = 0.f, w = 0.f;
    constexpr float LOG2E = 1.4426950408889634f;
    const int steps = p.group / STEP;  // of a group
    auto group_at = [&](int g) { return cta0 + static_cast<int64_t>(g) * p.group + lane * N; };
    auto live = [&](int g) { return g < p.groups && cta0 + static_cast<int64_t>(g) * p.group < end; };
    Vec<T> a, b;
    if (live(warp)) {
        a = load(group_at(warp));
        b = load(group_at(warp) + 32 * N);
    }
    for (int g = warp; g < p.groups; g += WARPS) {
        unsigned best = 0;
        if (live(g))
            for (int i = 0; i < steps; ++i) {
                const Vec<T> va = a, vb = b;
                {  // the next loads
                    const bool same = i + 1 < steps;
                    const int ng = same ? g : g + WARPS;
                    if (live(ng)) {
                        const int64_t at = group_at(ng) + (same ? (i + 1) * STEP : 0);
                        a = load(at);
                        b = load(at + 32 * N);
                    }
                }
                const unsigned ta = order_of(va.top()), tb = order_of(vb.top());
                if (p.fine) {
                    s_top[g * 64 + lane] = ta;
                    s_top[g * 64 + 32 + lane] = tb;
                }
                const unsigned top = __reduce_max_sync(0xffffffffu, max(ta, tb));
                best = max(best, top);
                if (top <= ORDER_NONE || top >= ORDER_INF) continue;  // nothing to add; NaN and +inf show in the maximum
                const float t = value_of(top);
                if (t > m) {
                    const float d = m - t, f = ex2(d * LOG2E);  // m = -inf: f = 0 and nothing was added
                    w = z > 0.f ? f * fmaf(d, z, w) : 0.f;
                    z *= f;
                    m = t;
                }
#pragma unroll
                for (int k = 0; k < 2 * N; ++k) {
                    const float d = fmaxf((k < N ? va[k] : vb[k - N]) - m, -1e30f);  // -inf: exp is 0, and 0 times it
                    const float e = ex2(d * LOG2E);
                    z += e;
                    w = fmaf(d, e, w);
                }
            }
        if (lane == 0 && !p.fine) s_top[g] = best;
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, k);
        w += __shfl_xor_sync(0xffffffffu, w, k);
    }
    if (lane == 0) {
        s_sum[warp][0] = m;
        s_sum[warp][1] = z;
        s_sum[warp][2] = w;
    }
    __syncthreads();
    // Joins (m, z, w) triples; the order is fixed.
    auto join = [&](float &m0, float &z0, float &w0, float m1, float z1, float w1) {
        const float t = fmaxf(m0, m1);
        if (t == -INFINITY) return;
        const float d0 = fmaxf(m0 - t, -1e30f), d1 = fmaxf(m1 - t, -1e30f);
        const float f0 = ex2(d0 * LOG2E), f1 = ex2(d1 * LOG2E);
        w0 = f0 * fmaf(d0, z0, w0) + f1 * fmaf(d1, z1, w1);
        z0 = z0 * f0 + z1 * f1;
        m0 = t;
    };
    if (threadIdx.x == 0) {
        float m0 = -INFINITY, z0 = 0.f, w0 = 0.f;
        for (int i = 0; i < WARPS; ++i) join(m0, z0, w0, s_sum[i][0], s_sum[i][1], s_sum[i][2]);
        s_row[0] = m0;
        s_row[1] = z0;
        s_row[2] = w0;
    }
    // ---- rank 0 has the row's sums and groups ---------------------------------------------------------
    const unsigned *tops = s_top;
    const int all = p.fine ? min(p.groups * 64, static_cast<int>((end + N - 1) / N)) : p.groups * p.cluster;
    const int group = p.fine ? N : p.group;
    if (p.cluster > 1) {
        ptx::cluster_sync();
        if (rank == 0) {
            for (int i = threadIdx.x; i < all; i += THREADS) {
                const uint32_t at = ptx::map_shared_rank(ptx::smem_u32(&s_top[i % p.groups]), i / p.groups);
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(s_all[i]) : "r"(at) : "memory");
            }
            if (threadIdx.x == 0)
                for (int r = 1; r < p.cluster; ++r) {
                    float v[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        const uint32_t at = ptx::map_shared_rank(ptx::smem_u32(&s_row[i]), r);
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[i]) : "r"(at) : "memory");
                    }
                    join(s_row[0], s_row[1], s_row[2], v[0], v[1], v[2]);
                }
            tops = s_all;
        }
        ptx::cluster_sync();  // the other CTAs' shared memory has been read
        if (rank != 0) return;
    }
    if (threadIdx.x == 0) {
        s_count = 0;
        s_sel_n = 0;
    }
    __syncthreads();
    unsigned most = 0;
    for (int i = threadIdx.x; i < all; i += THREADS) most = max(most, tops[i]);
    const bool nan = __syncthreads_or(most >= ORDER_INF);
    const float top = s_row[0], zz = s_row[1], ww = s_row[2];
    const bool empty = top == -INFINITY && !nan;
    const float log_z = logf(zz), none = __int_as_float(0x7fffffff);
    auto lp = [&](float v) { return nan ? none : empty ? -INFINITY : (v - top) - log_z; };
    if (threadIdx.x == 0) {
        p.entropy[row] = nan ? none : empty ? 0.f : log_z - ww / zz;
        if (p.tokens) {
            const int64_t t = p.tokens[row];
            const bool in = t >= 0 && t < p.V;
            if (!in) report_status(LSE_ERR_INVALID_ARG);
            p.logprob[row] = in ? lp(to_float(x[t])) : none;
        }
    }
    if (p.k == 0) return;

    // ---- the first k groups by (maximum, index) -------------------------------------------------------
    const int want = min(p.k, all);
    // a T that `want` groups reach (and so k logits), the largest or one with no group's maximum between;
    // 0 where there are no k groups
    unsigned lo = 0, hi = want < p.k ? 0u : 0xffffffffu;  // count(>= lo) >= want
    int reach = all;
    while (lo < hi) {
        const unsigned mid = lo + (hi - lo) / 2 + 1;
        int n = 0;
        for (int i0 = 0; i0 < all; i0 += THREADS) n += __syncthreads_count(i0 + threadIdx.x < all && tops[i0 + threadIdx.x] >= mid);
        if (n >= want) {
            lo = mid;
            reach = n;
            if (n == want) break;  // any threshold between gives the same groups
        } else {
            hi = mid - 1;
        }
    }
    if (warp == 0) {  // those above T, then those at T from the lowest index on
        int above = 0;
        for (int i0 = 0; i0 < all; i0 += 32) above += __popc(__ballot_sync(0xffffffffu, i0 + lane < all && tops[i0 + lane] > lo));
        int level = reach == want ? want : want - above;  // groups at T that still fit (all of them when the count is exact)
        int n = 0;
        for (int i0 = 0; i0 < all; i0 += 32) {
            const unsigned o = i0 + lane < all ? tops[i0 + lane] : 0u;
            const bool in = i0 + lane < all && o >= lo, at = in && o == lo;
            const unsigned eq = __ballot_sync(0xffffffffu, at);
            const bool take = in && (!at || __popc(eq & ((1u << lane) - 1u)) < level);
            const unsigned yes = __ballot_sync(0xffffffffu, take);
            if (take) s_sel[n + __popc(yes & ((1u << lane) - 1u))] = i0 + lane;
            n += __popc(yes);
            level -= __popc(eq & yes);
        }
        if (lane == 0) s_sel_n = n;
    }
    __syncthreads();
    const int sel_n = s_sel_n;
    // Keys of the logits of the selected groups: a warp's 16 bytes a lane at a time, or a lane's own (fine).
    auto visit = [&](auto f) {
        for (int s = p.fine ? threadIdx.x : warp; s < sel_n; s += p.fine ? THREADS : WARPS) {
            const int64_t g0 = static_cast<int64_t>(s_sel[s]) * group;  // (ranks' groups follow one another)
            for (int64_t at = g0 + (p.fine ? 0 : lane * N); at < min(g0 + group, end); at += 32 * N) {
                const Vec<T> v = load(at);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int64_t i = at + k - shift;
                    if (i >= 0 && i < p.V) f((static_cast<unsigned long long>(order_of(v[k])) << 32) | (0x7fffffffu - static_cast<unsigned>(i)));
                }
            }
        }
    };
    visit([&](unsigned long long key) {
        if ((key >> 32) >= lo) {
            const int at = atomicAdd(&s_count, 1);
            if (at < CANDIDATES) s_key[at] = key;
        }
    });
    __syncthreads();
    auto store = [&](int at, unsigned long long key) {
        const int64_t i = row * static_cast<int64_t>(p.k) + at;
        p.top_id[i] = 0x7fffffffu - static_cast<unsigned>(key);
        p.top_logprob[i] = lp(value_of(static_cast<unsigned>(key >> 32)));
    };
    const int count = s_count;
    if (count <= CANDIDATES) {
        for (int i = threadIdx.x; i < count; i += THREADS) {
            const unsigned long long key = s_key[i];
            int before = 0;
            for (int j = 0; j < count; ++j) before += s_key[j] > key;
            if (before < p.k) store(before, key);
        }
        return;
    }
    // Many logits reach T (equal ones, or a group full of large ones): one alternative a round.
    unsigned long long last = ~0ull;
    for (int r = 0; r < p.k; ++r) {
        unsigned long long best = 0;
        visit([&](unsigned long long key) {
            if (key < last && key > best) best = key;
        });
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, k));
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) best = max(best, s_best[i]);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) store(r, best);
    }
}

}  // namespace logprobs
}  // namespace lse
