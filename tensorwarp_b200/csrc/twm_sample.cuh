// twm_sample.cuh — one token of every row of logits: temperature, top-k, top-p, min-p (include/twm_serve.h).
//
// A row belongs to a cluster of CTAs, each with a slice of it in shared memory: logits are read from memory once, whatever cuts are asked for.
// Nothing is sorted.  The kept tokens are the head of an order, so all cuts come down to one key and how many of the tokens equal to it are
// kept; that border is found by histograms, narrowing in on the bin it lies in:
//   level 0   bins of 1/8 octave of weight below the largest logit's, 512 of them (what is beyond, 2^-64, is one more bin);
//   then      512 equal parts, as ordered integers, of the logits of the bin that the border lies in, and of the part again;
// and once 32 tokens or fewer are left they are ordered by one warp.  Where those of level 0's bin and all ahead of it are 128 at most, as for a small
// top-k or a sharp row, they go to the first CTA, which orders them and does the rest alone.  Which logits a bin of level 0 has is found by searching its ends, so that
// all passes but the first only compare.  A bin holds its number of tokens and its mass.  Within a bin weights are
// within 2^(1/8) of its largest W: mass = W (count - sum of delta), delta = 1 - w / W in fixed point, so that both are integer sums, the
// same in any order: the result does not depend on which thread comes first.
// Then running sums, by index, of the kept weights find the token.
// Bound by latency, for few rows and for many.  250 rows of 152064 take 207 us (152 MB read, 0.73 TB/s): seven waves of slices, of whose 26 us the load
// has three, shared atomics and the other passes over shared memory fourteen, cluster barriers the rest; 64 rows of 32768 take 24 us.  One row takes 14 us:
// of 25 500 clocks the first CTA's ordering of the last 128 tokens or fewer has 7200, the join of the histograms 3900, the histogram 2900, settings
// and start 2200, search and scan 2000, the draw 1500; five cluster barriers, the start's among them.
#pragma once

#include <algorithm>

#include <cuda_bf16.h>

#include "../../include/twm_serve.h"
#include "twm_common.cuh"

namespace twm {
namespace sample {

__device__ __forceinline__ float logit_f32(float v) { return v; }
__device__ __forceinline__ float logit_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float logit_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// NaN as -inf, both zeros alike
__device__ __forceinline__ float plain(float v) { return v == v ? v + 0.0f : -INFINITY; }
// numbers in the order of unsigned integers
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = THREADS, MAX_CTAS = 16, FEW = 32;
constexpr int ALL = 128;                 // tokens that the first CTA orders by itself
constexpr int MAX_SLICE = 40960;         // logits of a CTA in shared memory; what is beyond is read again

__device__ __forceinline__ void st_cluster_u32(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void st_cluster_u64(uint32_t at, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t at)
{
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// Weights below the largest logit's: exponents in octaves, the factor in two parts so that a weight is good to the last bits that ex2 has.
struct Weights {
    float top, hi, lo;
    __device__ __forceinline__ void set(float mx, double temperature)
    {
        const double c = fmin(1.4426950408889634 / temperature, 1e30);
        top = mx;
        hi = (float)c;
        lo = (float)(c - (double)hi);
    }
    __device__ __forceinline__ float of_finite(float v) const           // with a finite largest logit
    {
        const float d = v - top, x = d * hi, rest = fmaf(d, lo, fmaf(d, hi, -x));
        float y;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
        return x > -140.0f ? fmaf(y, rest * 0.69314718f, y) : 0.0f;
    }
    __device__ __forceinline__ float of(float v) const { return v == top ? 1.0f : of_finite(v); }
};

__device__ __forceinline__ uint32_t count_cluster(uint32_t at)          // adds one to a counter and gives what it was
{
    uint32_t v;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(v) : "r"(at) : "memory");
    return v;
}

struct Shared {
    uint32_t count[BINS], delta[BINS];                   // this CTA's, as it counts
    uint32_t all_count[BINS];                            // the cluster's
    unsigned long long all_delta[BINS];
    uint32_t part_count[THREADS];
    unsigned long long part_delta[THREADS];
    uint32_t warp_u32[WARPS];
    double warp_f64[WARPS];
    uint32_t cta_max[MAX_CTAS];
    uint32_t ends[2];                                    // the keys at which level 0's bin and the next one begin
    uint32_t cta_ties[MAX_CTAS];
    unsigned long long cta_above[MAX_CTAS];
    uint32_t list_n[2], list[2][FEW];                    // the last tokens of top-k's border, of top-p's
    uint32_t own_n;                                      // the slice's logits in the border's bin, if a thread has one at most
    float own[THREADS];
    uint32_t all_n, all_key[ALL], all_index[ALL];        // the first CTA's: all tokens down to the end of the border's bin
    uint32_t key[ALL], index[ALL], kept;                 // ... in order
    unsigned long long weight[ALL];
    uint32_t found_bin, found_count, found_over;
    double found_over_mass;
    uint32_t cut, ties;
    double cut_mass;
};

// 2^(-i / 8)
__device__ __constant__ double c_octave[8] = {1.0, 0.91700404320467123174, 0.84089641525371454303, 0.77110541270397041183, 0.70710678118654752440,
                                              0.64841977732550483296, 0.59460355750136053336, 0.54525386633262882960};
__device__ __forceinline__ double octave_part(int i) { return c_octave[i & 7] * __longlong_as_double((long long)(1023 - (i >> 3)) << 52); }

// counts and masses ahead of this thread's bin, and of all
struct Scan { uint32_t before, all; double mass_before, mass_all; };
__device__ __forceinline__ Scan scan(Shared& sh, uint32_t c, double m)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t uc = c;
    double um = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t xc = __shfl_up_sync(0xffffffffu, uc, o);
        const double xm = __shfl_up_sync(0xffffffffu, um, o);
        if (lane >= o) { uc += xc; um += xm; }
    }
    __syncthreads();
    if (lane == 31) { sh.warp_u32[warp] = uc; sh.warp_f64[warp] = um; }
    __syncthreads();
    // every warp adds up the warps' sums, a lane each
    uint32_t tc = lane < WARPS ? sh.warp_u32[lane] : 0u;
    double tm = lane < WARPS ? sh.warp_f64[lane] : 0.0;
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
        const uint32_t xc = __shfl_up_sync(0xffffffffu, tc, o);
        const double xm = __shfl_up_sync(0xffffffffu, tm, o);
        if (lane >= o) { tc += xc; tm += xm; }
    }
    Scan s;
    s.all = __shfl_sync(0xffffffffu, tc, WARPS - 1);
    s.mass_all = __shfl_sync(0xffffffffu, tm, WARPS - 1);
    const uint32_t bc = __shfl_sync(0xffffffffu, tc, (warp + 31) & 31), xc = __shfl_up_sync(0xffffffffu, uc, 1);
    const double bm = __shfl_sync(0xffffffffu, tm, (warp + 31) & 31), xm = __shfl_up_sync(0xffffffffu, um, 1);
    s.before = (warp ? bc : 0u) + (lane ? xc : 0u);
    s.mass_before = (warp ? bm : 0.0) + (lane ? xm : 0.0);
    return s;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2)
sample_kernel(const __grid_constant__ twm_sample_args a, int slice, int ctas)
{
    extern __shared__ __align__(16) float vals[];
    __shared__ Shared sh;
    cluster_started();
    pdl_launch_dependents();
    const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = a.vocab, n0 = min(n, rank * slice), ns = min(n - n0, slice);
    for (int i = tid; i < BINS; i += THREADS) sh.count[i] = sh.delta[i] = 0;
    if (tid < 2) sh.list_n[tid] = 0;
    if (tid == 0) sh.all_n = 0;
    pdl_wait_prior_grids();
    const T* logits = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld + n0;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    const float random = a.random[a.step ? min(max(a.step[0], 0), a.random_count - 1) : row];

    // ---- the slice into shared memory, and its largest logit ----
    const int held = min(ns, MAX_SLICE);
    float mx = -INFINITY;
    constexpr int V = 16 / sizeof(T);
    const int vecs = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 ? held / V : 0;
    for (int i = tid; i < vecs; i += THREADS) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(logits) + i);
        T x[V];
        *reinterpret_cast<uint4*>(x) = u;
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const float4 f = make_float4(plain(logit_f32(x[j])), plain(logit_f32(x[j + 1])), plain(logit_f32(x[j + 2])), plain(logit_f32(x[j + 3])));
            mx = fmaxf(mx, fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)));
            *reinterpret_cast<float4*>(vals + i * V + j) = f;
        }
    }
    for (int i = vecs * V + tid; i < ns; i += THREADS) {
        const float f = plain(logit_f32(logits[i]));
        mx = fmaxf(mx, f);
        if (i < held) vals[i] = f;
    }
    const int quads = (held + 3) / 4;
    if (tid < 4 * quads - held) vals[held + tid] = NAN;  // compares false with everything
    auto at = [&](int i) { return i < held ? vals[i] : plain(logit_f32(logits[i])); };
    auto each = [&](auto f) {
        for (int i = tid; i < quads; i += THREADS) {
            const float4 q = reinterpret_cast<const float4*>(vals)[i];
            f(q.x); f(q.y); f(q.z); f(q.w);
        }
        for (int i = held + tid; i < ns; i += THREADS) f(plain(logit_f32(logits[i])));
    };
    uint32_t key = __reduce_max_sync(0xffffffffu, order_of(mx));
    if (lane == 0) sh.warp_u32[warp] = key;
    __syncthreads();
    cluster_wait_started();
    if (tid < ctas) {
        key = 0;
        for (int w = 0; w < WARPS; ++w) key = max(key, sh.warp_u32[w]);
        st_cluster_u32(mapa_shared(smem_u32(&sh.cta_max[rank]), tid), key);
    }
    cluster_sync_all();
    key = 0;
    for (int c = 0; c < ctas; ++c) key = max(key, sh.cta_max[c]);
    mx = value_of(key);

    constexpr float ONE = 4398046511104.0f;              // 2^42
    auto answer = [&](int token, float prob) {           // by one thread of the cluster
        a.tokens[row] = token;
        if (a.prob) a.prob[row] = prob;
        if (a.step) {
            const int step = a.step[0];
            if (a.history && step >= 0 && step < a.history_capacity) a.history[step] = token;
            a.step[0] = step + 1;
            a.pos[0] += 1;
            a.len[0] += 1;
        }
    };
    // the lowest key that min_p keeps; at an infinite temperature all finite logits weigh 1, and the others nothing
    auto least_key = [&]() { return mp > 0.0f && t < INFINITY ? order_of(__double2float_ru((double)mx + (double)t * log(fmin((double)mp, 1.0))) + 0.0f) : 0u; };

    uint32_t cut = 0, ties = 0x7fffffffu;                // kept: keys over cut, and the first `ties` of those that are cut
    Weights weights = {mx, 0.0f, 0.0f};
    const bool none = mx == -INFINITY, greedy = !(t > 0.0f);
    if (none || greedy) {
        cut = key;
        ties = 1;
    } else {
        weights.set(mx, (double)t);
        const bool need_k = k > 0 && k < n, need_p = p < 1.0f;
        if (need_k || need_p) {
            // a token's bin at level 0, or BINS; falls with rising logits
            const float scale8 = -8.0f * weights.hi;
            auto place_of = [&](float v) { return v == mx ? 0.0f : (v - mx) * scale8; };
            auto bin_of = [&](float v) { const float x = place_of(v); return x < (float)BINS ? (int)x : BINS; };
            // delta < 0.0831: a slice's sum of them fits 32 bits
            const float fixed = slice <= 24000 ? 2097152.0f : slice <= 48000 ? 1048576.0f : 524288.0f;
            const double unit = 1.0 / (double)fixed;
            auto count = [&](int bin, float delta) {
                atomicAdd(&sh.count[bin], 1u);
                const uint32_t d = __float_as_uint(fmaf(delta, fixed, 8388608.0f)) - 0x4b000000u;        // the nearest integer
                if (d) atomicAdd(&sh.delta[bin], d);
            };
            // The cluster's histogram from those of its CTAs: each CTA adds up a share of the bins, every thread of one CTA's, and tells all.
            auto join = [&]() {
                cluster_sync_all();
                if (ctas == 1) {
                    sh.all_count[tid] = sh.count[tid];
                    sh.all_delta[tid] = sh.delta[tid];
                    sh.count[tid] = sh.delta[tid] = 0;       // the next ones to write there come behind a barrier
                    return;
                }
                const int bins = BINS / ctas, b = tid % bins, g = tid / bins, mine = rank * bins + b;
                sh.part_count[tid] = ld_cluster_u32(mapa_shared(smem_u32(&sh.count[mine]), g));
                sh.part_delta[tid] = ld_cluster_u32(mapa_shared(smem_u32(&sh.delta[mine]), g));
                __syncthreads();
                uint32_t c = 0;
                unsigned long long d = 0;
                for (int x = b; x < BINS; x += bins) { c += sh.part_count[x]; d += sh.part_delta[x]; }
                st_cluster_u32(mapa_shared(smem_u32(&sh.all_count[mine]), g), c);
                st_cluster_u64(mapa_shared(smem_u32(&sh.all_delta[mine]), g), d);
                cluster_sync_all();
                sh.count[tid] = sh.delta[tid] = 0;
            };
            // level 0; 1 - 2^(-y/8) = 1 - e^-z by its series, z < 0.0867
            auto put = [&](float x) {
                if (x < (float)BINS) {
                    const float whole = __fadd_rz(x, 8388608.0f);                // 2^23 + the bin
                    const float z = (x - (whole - 8388608.0f)) * (0.69314718f / 8.0f);
                    count((int)(__float_as_uint(whole) - 0x4b000000u), z * fmaf(z, fmaf(z, fmaf(z, -1.0f / 24.0f, 1.0f / 6.0f), -0.5f), 1.0f));
                }
            };
            if (mx < INFINITY) each([&](float v) { put((v - mx) * scale8); });
            else each([&](float v) { put(place_of(v)); });
            join();
            const uint32_t c0 = sh.all_count[tid];
            const double m0 = octave_part(tid) * ((double)c0 - (double)sh.all_delta[tid] * unit);
            const Scan first = scan(sh, c0, m0);
            double mass = first.mass_all;                    // of what top-k keeps

            // All tokens from key `lo` on, n of them, to the first CTA, which orders them by value and index: top-k, top-p and min-p all keep a head of
            // that order.  A token's running sum is that of the kept ones with lower indexes.
            auto finish_alone = [&](uint32_t lo, uint32_t n_all, bool need_k, double mass) {
                const float f_lo = value_of(lo);
                const uint32_t to_n = mapa_shared(smem_u32(&sh.all_n), 0), to_key = mapa_shared(smem_u32(sh.all_key), 0), to_index = mapa_shared(smem_u32(sh.all_index), 0);
                auto offer = [&](float v, int i) {
                    if (v >= f_lo) {
                        const uint32_t slot = count_cluster(to_n);
                        if (slot < ALL) { st_cluster_u32(to_key + 4 * slot, order_of(v)); st_cluster_u32(to_index + 4 * slot, (uint32_t)(n0 + i)); }
                    }
                };
                for (int i = tid; i < quads; i += THREADS) {
                    const float4 q = reinterpret_cast<const float4*>(vals)[i];
                    if (fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) >= f_lo) { offer(q.x, 4 * i); offer(q.y, 4 * i + 1); offer(q.z, 4 * i + 2); offer(q.w, 4 * i + 3); }
                }
                for (int i = held + tid; i < ns; i += THREADS) offer(plain(logit_f32(logits[i])), i);
                cluster_sync_all();
                if (rank != 0) return;
                const int m = (int)min(n_all, (uint32_t)ALL);
                if (tid < m) {
                    const uint32_t mine = sh.all_key[tid], index = sh.all_index[tid];
                    int place = 0;
                    for (int j = 0; j < m; ++j) place += sh.all_key[j] > mine || (sh.all_key[j] == mine && sh.all_index[j] < index);
                    sh.key[place] = mine;
                    sh.index[place] = index;
                }
                __syncthreads();
                if (warp == 0) {
                    constexpr int EACH = ALL / 32;
                    float w[EACH];
                    double upto = 0.0;
                    const int n_k = need_k ? min(m, k) : m;
#pragma unroll
                    for (int j = 0; j < EACH; ++j) {
                        const int i = lane * EACH + j;
                        w[j] = i < m ? weights.of(value_of(sh.key[i])) : 0.0f;
                        if (i < n_k) upto += (double)w[j];
                        if (i < m) sh.weight[i] = __float2ull_rn(w[j] * ONE);
                    }
                    const double own = upto;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double x = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += x;
                    }
                    if (need_k) mass = __shfl_sync(0xffffffffu, upto, 31);
                    const double want = (double)p * mass;
                    const uint32_t least = least_key();
                    double before = upto - own;
                    int kept = 0;
#pragma unroll
                    for (int j = 0; j < EACH; ++j) {
                        const int i = lane * EACH + j;
                        kept += i < n_k && (i == 0 || ((!need_p || before < want) && sh.key[i] >= least));
                        before += (double)w[j];
                    }
                    kept = __reduce_add_sync(0xffffffffu, kept);
                    if (lane == 0) sh.kept = kept;
                }
                __syncthreads();
                const int kept = (int)sh.kept;
                if (tid < kept) {
                    const uint32_t index = sh.index[tid];
                    unsigned long long before = 0, total = 0;
                    for (int j = 0; j < kept; ++j) {
                        total += sh.weight[j];
                        if (sh.index[j] < index) before += sh.weight[j];
                    }
                    const unsigned long long target = min((unsigned long long)(fmin(fmax((double)random, 0.0), 1.0) * (double)total), total - 1);
                    if (before <= target && target < before + sh.weight[tid])
                        answer((int)index, (float)((double)weights.of(value_of(sh.key[tid])) * (double)ONE / (double)total));
                }
            };

            for (int what = need_k ? 0 : 1; what <= (need_p ? 1 : 0); ++what) {
                const double want = fmax((double)p * mass, 1e-30);       // of mass, for top-p
                // The bin with the border, from this thread's: the first whose end reaches what is wanted; the last one with tokens if rounding keeps
                // all from it.  Its number, tokens and mass, and those ahead of it.
                auto find = [&](uint32_t over, double over_mass, uint32_t x, double y, const Scan& s, uint32_t beyond) {
                    if (tid == 0) sh.found_bin = BINS;
                    __syncthreads();
                    if (x > 0 && (what == 0 ? over + s.before + x >= (uint32_t)k : over_mass + s.mass_before + y >= want)) atomicMin(&sh.found_bin, (uint32_t)tid);
                    __syncthreads();
                    if (what == 1 && sh.found_bin == BINS) {
                        __syncthreads();
                        if (x > 0 && s.before + x == s.all) sh.found_bin = tid;              // one thread's alone
                        __syncthreads();
                    }
                    const uint32_t b = sh.found_bin;
                    if (b == tid) {
                        sh.found_count = x;
                        sh.found_over = over + s.before;
                        sh.found_over_mass = over_mass + s.mass_before;
                    }
                    if (b == BINS && tid == 0) {             // top-k's border lies beyond the bins
                        sh.found_count = beyond;
                        sh.found_over = over + s.all;
                        sh.found_over_mass = over_mass + s.mass_all;
                    }
                    __syncthreads();
                };
                find(0, 0.0, c0, m0, first, (uint32_t)n - first.all);
                const int bin = (int)sh.found_bin;
                uint32_t left = sh.found_count, over = sh.found_over;
                double over_mass = sh.found_over_mass;
                // the logits that are left, as keys: from the end of the next bin to that of this one, each found by a warp
                const uint32_t lowest = order_of(-INFINITY);
                if (warp < 2) {
                    uint32_t from = lowest, to = key;            // the largest key whose bin is `bin` (or the next one) or behind it
                    const int b = bin + warp;
                    if (b == 0) from = key;
                    else if (b > BINS) from = lowest - 1;
                    else {
                        // next to where the arithmetic without rounding has it, if it is there
                        const uint32_t near = order_of(fminf(fmaxf(mx + (float)b / scale8, -3.4e38f), mx)), below = near - min(near - lowest, 256u);
                        if (near > lowest + 512 && bin_of(value_of(below)) >= b && (near + 256 > key || bin_of(value_of(near + 256)) < b)) {
                            from = below;
                            to = min(key, near + 255);
                        }
                        while (from < to) {
                            const uint32_t step = (to - from) / 32 + 1;
                            const uint32_t mine = from + (lane + 1) * step;
                            const unsigned int yes = __ballot_sync(0xffffffffu, mine > from && mine <= to && bin_of(value_of(mine)) >= b);
                            const uint32_t next = from + __popc(yes) * step;
                            to = min(to, next + (step - 1));
                            from = next;
                        }
                    }
                    if (lane == 0) sh.ends[warp] = from;
                }
                __syncthreads();
                uint32_t hi = sh.ends[0], lo = sh.ends[1] + 1;
                if (bin < BINS && over + left <= ALL && !(what == 1 && need_k)) {
                    finish_alone(lo, over + left, need_k, mass);
                    return;
                }
                // the logits that are left of this slice, one a thread, where there are so few
                const bool many = left > FEW && lo < hi;
                if (many) {
                    if (tid == 0) sh.own_n = 0;
                    __syncthreads();
                    const float f_lo = value_of(lo), f_hi = value_of(hi);
                    each([&](float v) {
                        if (v >= f_lo && v <= f_hi) {
                            const uint32_t slot = atomicAdd(&sh.own_n, 1u);
                            if (slot < THREADS) sh.own[slot] = v;
                        }
                    });
                    __syncthreads();
                }
                const uint32_t own_n = many ? sh.own_n : THREADS + 1;
                auto each_left = [&](auto f) {                   // f for those of [lo, hi]
                    const float f_lo = value_of(lo), f_hi = value_of(hi);
                    if (own_n <= THREADS) {
                        if (tid < own_n && sh.own[tid] >= f_lo && sh.own[tid] <= f_hi) f(sh.own[tid]);
                    } else {
                        each([&](float v) { if (v >= f_lo && v <= f_hi) f(v); });
                    }
                };
                while (left > FEW && lo < hi) {
                    const int shift = max(0, 23 - __clz(hi - lo));               // (hi - lo) >> shift < 512
                    const float w_top = weights.of(value_of(hi)), back = 1.0f / w_top;
                    each_left([&](float v) {                     // beyond the bins mass does not count
                        count((int)((hi - order_of(v)) >> shift), bin < BINS ? fmaxf(fmaf(-weights.of(v), back, 1.0f), 0.0f) : 0.0f);
                    });
                    join();
                    const uint32_t x = sh.all_count[tid];
                    const double y = bin < BINS ? (double)w_top * ((double)x - (double)sh.all_delta[tid] * unit) : 0.0;
                    find(over, over_mass, x, y, scan(sh, x, y), 0);
                    const uint32_t b = sh.found_bin;
                    left = sh.found_count;
                    over = sh.found_over;
                    over_mass = sh.found_over_mass;
                    hi -= b << shift;
                    lo = max(lo, hi - min(hi, (1u << shift) - 1u));
                }
                uint32_t border, border_ties;
                if (left > FEW) {                            // equal ones only
                    __syncthreads();                         // all have read what the last `find` left, which that of the next pass resets
                    const double w = (double)weights.of(value_of(lo));
                    border = lo;
                    border_ties = what == 0 ? (uint32_t)k - over : w > 0.0 ? (uint32_t)fmin(fmax(ceil((want - over_mass) / w), 1.0), (double)left) : left;
                    mass = over_mass + (double)border_ties * w;
                } else {
                    // the last ones, put in order by a warp of every CTA
                    each_left([&](float v) {
                        const uint32_t slot = atomicAdd(&sh.list_n[what], 1u);
                        if (slot < FEW) sh.list[what][slot] = order_of(v);
                    });
                    cluster_sync_all();
                    if (warp == 0) {
                        // lane x takes the x-th of the CTAs' lists, one behind another
                        const int m = lane < ctas ? (int)ld_cluster_u32(mapa_shared(smem_u32(&sh.list_n[what]), lane)) : 0;
                        int upto_cta = m;
#pragma unroll
                        for (int o = 1; o < MAX_CTAS; o <<= 1) {
                            const int x = __shfl_up_sync(0xffffffffu, upto_cta, o);
                            if (lane >= o) upto_cta += x;
                        }
                        int from = 0, base = 0;
                        for (int c = 0; c < ctas; ++c) {
                            const int x = __shfl_sync(0xffffffffu, upto_cta, c);
                            if (lane >= x) { from = c + 1; base = x; }
                        }
                        uint32_t mine = 0;
                        if (lane < (int)left) mine = ld_cluster_u32(mapa_shared(smem_u32(&sh.list[what][lane - base]), from));
                        int place = 0;
                        for (int j = 0; j < (int)left; ++j) {
                            const uint32_t x = __shfl_sync(0xffffffffu, mine, j);
                            place += x > mine || (x == mine && j < lane);
                        }
                        if (lane >= (int)left) place = lane;
                        sh.part_count[place] = mine;
                        __syncwarp();
                        mine = sh.part_count[lane];                              // falling; lanes from `left` on have none
                        const double w = lane < (int)left ? (double)weights.of(value_of(mine)) : 0.0;
                        double upto = w;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const double x = __shfl_up_sync(0xffffffffu, upto, o);
                            if (lane >= o) upto += x;
                        }
                        const bool kept = lane < (int)left && (what == 0 ? over + lane < (uint32_t)k : lane == 0 || over_mass + (upto - w) < want);
                        const unsigned int who = __ballot_sync(0xffffffffu, kept);
                        const int last = 31 - __clz(who | 1u);                   // a head of the order
                        const uint32_t of_last = __shfl_sync(0xffffffffu, mine, last);
                        const unsigned int same = __ballot_sync(0xffffffffu, kept && mine == of_last && lane <= last);
                        const double sum = __shfl_sync(0xffffffffu, upto, last);
                        if (lane == 0) { sh.cut = of_last; sh.ties = __popc(same); sh.cut_mass = over_mass + sum; }
                    }
                    __syncthreads();
                    border = sh.cut;
                    border_ties = sh.ties;
                    mass = sh.cut_mass;
                }
                if (border > cut) {                          // top-p's border may be rounded behind top-k's, which then stays
                    cut = border;
                    ties = border_ties;
                } else if (border == cut) {
                    ties = min(ties, border_ties);
                }
            }
        }
        const uint32_t least = least_key();
        if (least > cut) { cut = least; ties = 0x7fffffffu; }
    }

    // ---- running sums by index: neighbouring tokens a thread.  Weights as integers, 2^42 the largest:
    // the threads' sums add up exactly, in any order, so that exactly one thread has the token. ----
    const int per = 4 * (((ns + 4 * THREADS - 1) / (4 * THREADS)) | 1), i0 = min(ns, tid * per), i1 = min(ns, i0 + per);
    const float f_cut = cut < order_of(-INFINITY) ? -INFINITY : value_of(cut);       // all are over 0, but -inf weighs nothing
    float sum = 0.0f;                                    // of a thread's, in FP32, always in the same order
    uint32_t same = 0;
    auto walk = [&](auto weigh) {
        for (int i = i0; i < min(i1, held); i += 4) {        // an odd number of four each: no bank conflicts
            const float4 q = *reinterpret_cast<const float4*>(vals + i);
            weigh(q.x); weigh(q.y); weigh(q.z); weigh(q.w);
        }
        for (int i = max(i0, held); i < i1; ++i) weigh(plain(logit_f32(logits[i])));
    };
    if (mx < INFINITY) walk([&](float v) { if (v > f_cut) sum += weights.of_finite(v); same += v == f_cut; });
    else walk([&](float v) { if (v > f_cut) sum += weights.of(v); same += v == f_cut; });
    const unsigned long long above = __float2ull_rn(sum * ONE);
    unsigned long long upto = above;
    uint32_t same_upto = same;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
        const uint32_t y = __shfl_up_sync(0xffffffffu, same_upto, o);
        if (lane >= o) { upto += x; same_upto += y; }
    }
    __syncthreads();
    if (lane == 31) { sh.part_delta[warp] = upto; sh.part_count[warp] = same_upto; }
    __syncthreads();
    unsigned long long cta_above = 0;
    uint32_t cta_ties = 0;
    upto -= above;                                       // ahead of this thread
    same_upto -= same;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) { upto += sh.part_delta[w]; same_upto += sh.part_count[w]; }
        cta_above += sh.part_delta[w];
        cta_ties += sh.part_count[w];
    }
    if (tid < ctas) {
        st_cluster_u32(mapa_shared(smem_u32(&sh.cta_ties[rank]), tid), cta_ties);
        st_cluster_u64(mapa_shared(smem_u32(&sh.cta_above[rank]), tid), cta_above);
    }
    cluster_sync_all();
    unsigned long long total = 0;
    uint32_t all_ties = 0;
    for (int c = 0; c < ctas; ++c) {
        if (c < rank) { upto += sh.cta_above[c]; same_upto += sh.cta_ties[c]; }
        total += sh.cta_above[c];
        all_ties += sh.cta_ties[c];
    }
    const float w_cut = none ? 1.0f : weights.of(value_of(cut));
    const unsigned long long one_tie = __float2ull_rn(w_cut * ONE);
    total += one_tie * min(all_ties, ties);
    const unsigned long long target = min((unsigned long long)(fmin(fmax((double)random, 0.0), 1.0) * (double)total), total - 1);
    const unsigned long long begin = upto + one_tie * min(same_upto, ties), end = upto + above + one_tie * min(same_upto + same, ties);
    if (begin <= target && target < end) {
        float w = 0.0f;
        int i = i0;
        sum = 0.0f;
        for (;; ++i) {                                       // the same sums again, up to the token whose weight passes the target
            const float v = at(i);
            if (v > f_cut) sum += w = weights.of(v);
            else if (v == f_cut && same_upto < ties) { ++same_upto; w = w_cut; }
            if (upto + __float2ull_rn(sum * ONE) + one_tie * min(same_upto, ties) > target) break;
        }
        answer(n0 + i, (float)((double)w * (double)ONE / (double)total));
    }
}

// ---------------------------------------------------------------------------------------------------------- launch --

inline twm_status check(const twm_sample_args* a)
{
    if (!a || !a->logits || !a->random || !a->tokens || a->rows < 1 || a->rows > (1 << 26) || a->vocab < 1 || a->vocab > (1 << 20) || a->ld < a->vocab) return TWM_EINVAL;
    if (a->dtype != TWM_F32 && a->dtype != TWM_F16 && a->dtype != TWM_BF16) return TWM_EINVAL;
    if (a->step && (a->rows != 1 || a->random_count < 1 || !a->pos || !a->len || (a->history && a->history_capacity < 1))) return TWM_EINVAL;
    return reinterpret_cast<uintptr_t>(a->logits) & (a->dtype == TWM_F32 ? 3 : 1) ? TWM_EALIGN : TWM_OK;
}

// The CTAs of a row: slices of at most 24000 logits, of which two fit an SM, and where there are few rows as many more of them as `sms` SMs take at
// once, down to 2048 logits each (64 rows of 32768, two or four CTAs: 28.1 and 25.5 us; 250 rows of 152064 in slices of at most 12000, 24000 and 39000
// logits: 311, 207 and 253 us).
template <typename T>
cudaError_t launch_as(const twm_sample_args& a, int sms, int flags, cudaStream_t stream)
{
    const int most = 2 * sms / std::min(a.rows, 2 * sms);
    int ctas = 1;
    while (ctas < MAX_CTAS && (a.vocab > 24000L * ctas || (2 * ctas <= most && a.vocab > 2048L * ctas))) ctas *= 2;
    const int slice = (int)((((long)a.vocab + ctas - 1) / ctas + 15) / 16 * 16);
    static_assert(MAX_SLICE * 4 + sizeof(Shared) + 1024 < 227 * 1024, "shared memory of a CTA");
    auto* kernel = sample_kernel<T>;
    cudaError_t e;
    // both belong to the function and only ever get these values
    if ((e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SLICE * 4)) != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = 4 * (size_t)std::min(slice, MAX_SLICE);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = flags & TWM_FLAG_PDL ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, slice, ctas);
}
inline cudaError_t launch(const twm_sample_args& a, int sms, int flags, void* stream)
{
    if (a.dtype == TWM_F32) return launch_as<float>(a, sms, flags, (cudaStream_t)stream);
    return a.dtype == TWM_F16 ? launch_as<__half>(a, sms, flags, (cudaStream_t)stream) : launch_as<__nv_bfloat16>(a, sms, flags, (cudaStream_t)stream);
}

}  // namespace sample
}  // namespace twm
