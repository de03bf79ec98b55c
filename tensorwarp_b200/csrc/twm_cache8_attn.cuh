// twm_cache8_attn.cuh — softmax attention over the cache held in 8 bits.
#pragma once

#include "twm_cache8.cuh"

namespace twm {
namespace cache8 {

struct AttnArgs {
    Cache c;
    Rows r;
    __half* out;
    const __half* q;
    long ldo, ldq;
    int num_heads, window;       // window: INT_MAX = all
    float scale;
};

__device__ __forceinline__ float code_value(uint8_t code) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3))); }

// A warp a query and head, a key at a time, FP32.
constexpr int PLAIN_THREADS = 128;
template <int D>
__global__ void __launch_bounds__(PLAIN_THREADS)
attn_plain_kernel(const __grid_constant__ AttnArgs a)
{
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int seq = blockIdx.y, lane = threadIdx.x & 31;
    int w = blockIdx.x * (PLAIN_THREADS / 32) + (threadIdx.x >> 5);
    const int i = w / a.num_heads, head = w % a.num_heads;
    const Span sp = span_of(a.r, seq, a.c.capacity);
    if (a.r.start[seq] < 0) {                                   // out of the call: zeros
        const int row = a.r.row_start ? a.r.row_start[seq] + i : seq;
        const int end = a.r.row_start ? a.r.row_start[seq + 1] : seq + 1;
        if (row < 0 || row >= min(end, a.r.rows) || i >= a.r.max_rows) return;
        for (int d = lane; d < D; d += 32) a.out[(size_t)row * a.ldo + head * D + d] = __float2half_rn(0.0f);
        return;
    }
    if (i >= sp.n) return;
    const int h = head / (a.num_heads / a.c.kv_heads), pos = sp.pos + i, full = (sp.pos + sp.n) / BLOCK;
    const size_t at = (size_t)seq * a.c.kv_heads + h;
    float q[D / 32], o[D / 32];
    for (int d = 0; d < D / 32; ++d) { q[d] = __half2float(a.q[(size_t)(sp.row + i) * a.ldq + head * D + lane + d * 32]); o[d] = 0.0f; }
    float m = -INFINITY, l = 0.0f;
    for (int j = a.window > pos ? 0 : pos - a.window + 1; j <= pos; ++j) {
        const int b = j / BLOCK;
        float k[D / 32], v[D / 32], s = 0.0f;
        if (b < full) {
            const size_t src = (at * a.c.capacity + j) * D + lane, sc = at * (a.c.capacity / BLOCK) + b;
            for (int d = 0; d < D / 32; ++d) { k[d] = code_value(a.c.k[src + d * 32]) * a.c.k_scale[sc]; v[d] = code_value(a.c.v[src + d * 32]) * a.c.v_scale[sc]; }
        } else {
            const size_t src = ((at * 2 + (b & 1)) * BLOCK + j % BLOCK) * D + lane;
            for (int d = 0; d < D / 32; ++d) { k[d] = __half2float(a.c.k_tail[src + d * 32]); v[d] = __half2float(a.c.v_tail[src + d * 32]); }
        }
        for (int d = 0; d < D / 32; ++d) s = fmaf(q[d], k[d], s);
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.scale;
        const float top = fmaxf(m, s), before = m == -INFINITY ? 0.0f : expf(m - top), p = expf(s - top);
        m = top;
        l = l * before + p;
        for (int d = 0; d < D / 32; ++d) o[d] = fmaf(p, v[d], o[d] * before);
    }
    for (int d = 0; d < D / 32; ++d) a.out[(size_t)(sp.row + i) * a.ldo + head * D + lane + d * 32] = __float2half_rn(o[d] / l);
}

}  // namespace cache8
}  // namespace twm
