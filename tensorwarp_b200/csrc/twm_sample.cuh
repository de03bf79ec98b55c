// twm_sample.cuh — one token of every row of logits: temperature, top-k, top-p, min-p (include/twm_serve.h).
#pragma once

#include <cuda_bf16.h>

#include "../../include/twm_serve.h"
#include "twm_common.cuh"

namespace twm {
namespace sample {

__device__ __forceinline__ float logit_f32(float v) { return v; }
__device__ __forceinline__ float logit_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float logit_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Numbers in the order of unsigned integers: NaN as -inf, both zeros alike.
__device__ __forceinline__ uint32_t order_of(float v)
{
    v = v == v ? v + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

constexpr int THREADS = 1024;

template <typename T>
__global__ void __launch_bounds__(THREADS)
sample_kernel(const __grid_constant__ twm_sample_args a)
{
    __shared__ double red[32];
    __shared__ double prefix[THREADS + 1];
    __shared__ int s_token;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int row = blockIdx.x, tid = threadIdx.x, n = a.vocab;
    const T* logits = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
    auto total = [&](double v) {
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = v;
        __syncthreads();
        double t = 0;
        for (int w = 0; w < THREADS / 32; ++w) t += red[w];
        return t;
    };
    auto key = [&](int i) { return order_of(logit_f32(logits[i])); };
    // largest, first index of it
    __shared__ unsigned long long s_best;
    if (tid == 0) s_best = 0;
    __syncthreads();
    unsigned long long best = 0;
    for (int i = tid; i < n; i += THREADS) best = max(best, ((unsigned long long)key(i) << 32) | (0xffffffffu - (uint32_t)i));
    atomicMax(&s_best, best);
    __syncthreads();
    const uint32_t top = (uint32_t)(s_best >> 32);
    const int first = (int)(0xffffffffu - (uint32_t)s_best);
    const float mx = value_of(top);
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    float prob = 1.0f;
    int token = mx == -INFINITY ? 0 : first;
    if (t > 0.0f && mx != -INFINITY) {
        const double inv_t = 1.0 / (double)t;
        auto weight = [&](uint32_t k) {
            const float v = value_of(k);
            return v == mx ? 1.0 : mx == INFINITY || v == -INFINITY ? 0.0 : exp(((double)v - (double)mx) * inv_t);
        };
        // kept: keys over `cut`, and the first `ties` of those equal to it
        uint32_t cut = 0;
        double ties = n;
        const int k = a.top_k ? a.top_k[row] : 0;
        const float p = a.top_p ? a.top_p[row] : 1.0f, mp = fminf(a.min_p ? a.min_p[row] : 0.0f, 1.0f);
        // the largest key with measure(keys >= it) >= want, and what of the measure is over it
        auto search = [&](auto measure, double want, double& over) {
            uint32_t lo = 0;                                     // measure(>= 0) >= want
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t mid = lo | (1u << bit);
                double v = 0;
                for (int i = tid; i < n; i += THREADS) { const uint32_t x = key(i); if (x >= mid) v += measure(x); }
                if (total(v) >= want) lo = mid;
            }
            double v = 0;
            for (int i = tid; i < n; i += THREADS) { const uint32_t x = key(i); if (x > lo) v += measure(x); }
            over = total(v);
            return lo;
        };
        double mass = 0, over;
        if (k > 0 && k < n) {
            cut = search([](uint32_t) { return 1.0; }, k, over);
            ties = k - over;
        }
        if (p < 1.0f) {
            double v = 0;
            for (int i = tid; i < n; i += THREADS) { const uint32_t x = key(i); if (x > cut) v += weight(x); }
            mass = total(v);
            double same = 0;
            for (int i = tid; i < n; i += THREADS) same += key(i) == cut;
            same = total(same);
            if (same > 0) mass += fmin(same, ties) * weight(cut);
            const double want = fmax((double)p * mass, 1e-30);
            const uint32_t c = max(cut, search(weight, fmin(want, mass * 0.9999999999), over));
            if (c > cut || over >= want) ties = n;
            cut = c;
            ties = fmin(ties, fmax(1.0, ceil((want - over) / fmax(weight(cut), 1e-300))));
        }
        if (mp > 0.0f) {
            const double least = (double)mx + (double)t * log((double)mp);
            const float f = __double2float_ru(least);
            const uint32_t c = order_of(f);
            if (c > cut) { cut = c; ties = n; }
        }
        // contiguous ranges a thread: equal keys before it, then running sums
        const int per = (n + THREADS - 1) / THREADS, i0 = min(n, tid * per), i1 = min(n, i0 + per);
        auto scan = [&](double v) {                              // prefix[t] = sum of the threads before t
            __syncthreads();
            prefix[tid + 1] = v;
            __syncthreads();
            if (tid == 0) { prefix[0] = 0; for (int i = 0; i < THREADS; ++i) prefix[i + 1] += prefix[i]; }
            __syncthreads();
        };
        double same = 0;
        for (int i = i0; i < i1; ++i) same += key(i) == cut;
        scan(same);
        const double rank0 = prefix[tid];
        auto walk = [&](auto each) {
            double rank = rank0;
            for (int i = i0; i < i1; ++i) {
                const uint32_t x = key(i);
                if (x > cut || (x == cut && rank < ties)) each(i, weight(x));
                rank += x == cut;
            }
        };
        double sum = 0;
        walk([&](int, double w) { sum += w; });
        scan(sum);
        if (tid == 0) s_token = 0x7fffffff;
        __syncthreads();
        int u_at = row;
        if (a.step) u_at = min(max(a.step[0], 0), a.random_count - 1);
        const float u = a.random[u_at];
        const double all = prefix[THREADS], want = fmin(fmax(u, 0.0f), 1.0f) * all;
        double run = prefix[tid];
        int found = 0x7fffffff, lastw = -1;
        walk([&](int i, double w) { run += w; if (w > 0) lastw = i; if (found == 0x7fffffff && w > 0 && run > want) found = i; });
        if (found != 0x7fffffff) atomicMin(&s_token, found);
        __syncthreads();
        if (s_token == 0x7fffffff) {                             // random rounds up to the whole sum: the last one
            __syncthreads();
            if (tid == 0) s_token = -1;
            __syncthreads();
            if (lastw >= 0) atomicMax(&s_token, lastw);
            __syncthreads();
        }
        token = s_token;
        prob = (float)(weight(key(token)) / all);
    }
    if (tid == 0) {
        a.tokens[row] = token;
        if (a.prob) a.prob[row] = prob;
        if (a.step) {
            const int step = a.step[0];
            if (a.history && step >= 0 && step < a.history_capacity) a.history[step] = token;
            a.step[0] += 1;
            a.pos[0] += 1;
            a.len[0] += 1;
        }
    }
}

}  // namespace sample
}  // namespace twm
