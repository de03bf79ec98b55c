// twm_cache8_prompt.cuh — softmax attention of many rows over the cache held in 8 bits, on the 5th-generation tensor cores.
//
// A tile is 256 rows, two MMA tiles of 128, which share every unit of 64 keys and values; a CTA takes an equal run of all units (see
// twm_cache8_attn.cuh, also for the mathematics).
//   warp 12     TMA: the units' codes, into a ring.
//   warps 8-11  codes to FP16, exactly, into the swizzled layout the MMAs read (rows of 64 elements, 128 bytes); a unit of the tail is copied instead.
//               Lanes take four chunks of 16 codes of rows r and r ^ 5, so that neither the reads nor the writes meet in a bank.
//   warp 13     one thread issues tcgen05.mma: half by half the scores of unit u + 1, then P V of unit u (P from tensor memory), so that the halves are
//               not at their exponentials at once.
//   warps 0-7   thread = row: maximum, weights, sum; the reference of the exponents moves only when a factor would pass 2^15, and then the row's output is
//               scaled in tensor memory ahead of the unit's P V.  They bring the rows' queries to shared memory and store the results.
// Tensor memory: two score buffers of 64 columns and D of output for each half; the factors, FP16, overwrite the scores.
// Sharing a unit between two halves is what shared memory asks for: a unit costs 16 KB read and 32 KB written by the conversion and 64 KB read by
// each half's MMAs, 1400 clocks at 128 bytes each for 256 rows against 1024 of MMA and 1024 of exponentials; with 128 rows it would be 1800.
// A prompt of 4000 tokens of 28 heads takes 153 us, 748 TFLOP/s, about 2400 clocks a unit.  What bounds that is not settled: without exponentials it takes
// 151 us, without the conversion 145, without the scores' MMAs 152, without all three 109, which is more than the products and the loads
// need.  All fourteen warps have 128 registers a thread, and the rows' (D = 128) store 72 bytes of them.
// Both halves' scores first and both halves' products then took 159 us; sixteen warps, half a row each, 174.
#pragma once

#include "twm_cache8_attn.cuh"
#include "twm_gemm_tcw.cuh"

namespace twm {
namespace cache8 {

constexpr int PROMPT_THREADS = 448;
constexpr int PROMPT_EXTRA = 8;                                          // a tile's own time, in units (prompt of 4000: 4 153.9 us, 8 155.3, 12 161.9; 56 of 642: 98, 95, 91.5)
constexpr int PROMPT_LEAST = 4;                                          // units of a CTA at least (10 rows of 16 heads on 4 after 2024 tokens: 1 21.3 us, 4 18.3, 8 18.5)
template <int D>
struct Prompt {
    static constexpr int BOXES = D / 64;
    static constexpr int QBOX = 128 * 128, KBOX = BLOCK * 128;           // bytes of 64 elements of 128 rows, of a unit's keys
    static constexpr int RAW = 2 * BLOCK * D, RAWS = 3;                  // a unit's codes; units in the ring
    static constexpr int UNIT = 2 * BOXES * KBOX, UNITS = 3;             // ... as FP16
    static constexpr int TMEM = 512, HALF = 256, OUT = 128;              // columns: of all, of a half, where its output is
    static constexpr size_t SMEM = 1024 + 2 * BOXES * (size_t)QBOX + UNITS * (size_t)UNIT + RAWS * (size_t)RAW;
};

__device__ __forceinline__ uint64_t row_desc(uint32_t addr)             // K-major, 128-byte swizzle
{
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t value_desc(uint32_t addr, uint32_t box)      // columns contiguous, the next 64 in the next box
{
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(box >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// two FP32 operations at once
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 r, x, y, z;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return r;
}

// Whether a unit's values are all zeros.  Its scores are done, so that the values are there and stay; ahead of them the parity of `full` would not tell,
// since a half that a tile did not have comes to the next one ahead of the conversion.  A call, so that the loop around it keeps its registers (prompt of
// 4000: 152.7 us, 158.5 in line).
__device__ __noinline__ bool no_values(const uint4* values, int words, uint64_t* full, uint32_t parity, volatile int* abort_flag)
{
    tc::wait_uniform(full, parity, abort_flag);
    bool any = false;
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < words && !any; i += 32) {
        const uint4 v = values[i];
        any = __any_sync(0xffffffffu, ((v.x | v.y | v.z | v.w) & 0x7fff7fffu) != 0);
    }
    return !any;
}

template <int D>
__global__ void __launch_bounds__(PROMPT_THREADS, 1)
prompt_kernel(const __grid_constant__ AttnArgs a)
{
    using P = Prompt<D>;
    extern __shared__ uint8_t prompt_raw[];
    __shared__ uint64_t raw_full[P::RAWS], raw_empty[P::RAWS], unit_full[P::UNITS], unit_empty[P::UNITS], q_full, s_full[2][2], p_full[2][2], o_done[2][2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_without[8];                                // units of tiles that a warp of rows had no part in
    uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(prompt_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* units = qs + 2 * P::BOXES * P::QBOX;
    uint8_t* raws = units + P::UNITS * P::UNIT;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < P::RAWS; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 4); }
        for (int i = 0; i < P::UNITS; ++i) { mbar_init(&unit_full[i], 4); mbar_init(&unit_empty[i], 1); }
        mbar_init(&q_full, 8);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&s_full[x][0], 1);
            mbar_init(&s_full[x][1], 1);
            mbar_init(&p_full[x][0], 4);
            mbar_init(&p_full[x][1], 4);
            mbar_init(&o_done[x][0], 1);
            mbar_init(&o_done[x][1], 1);
        }
        s_abort = 0;
        for (int i = 0; i < 8; ++i) s_without[i] = 0;
        mbar_fence_init();
    }
    // tensor memory is asked for once the kernel before has given its own back: an allocation waits without a limit
    pdl_wait_prior_grids();
    const Deal deal = {a.num_heads / a.c.kv_heads, PROMPT_ROWS, a.window, PROMPT_EXTRA, PROMPT_LEAST};
    const Start start = find_start<PROMPT_THREADS>(a, deal, blockIdx.x, gridDim.x);
    if (start.out) zero_rows(a, D, blockIdx.x, gridDim.x, tid, PROMPT_THREADS);
    Walk w;
    if (!w.begin(a, deal, start)) {
        if (tid == 0) a.joins[blockIdx.x].parts = 0;
        return;
    }
    if (warp == 13) {
        tc::tmem_alloc(&s_tmem, P::TMEM);
        tc::tc_fence_before();
    }
    __syncthreads();
    tc::tc_fence_after();
    pdl_launch_dependents();
    volatile int* abort_flag = &s_abort;
    const uint32_t tmem = s_tmem;

    if (warp == 12) {
        if (lane == 0) {
            int i = 0;
            bool ok = true;
            do {
                const int held = (w.sp.pos + w.sp.n) / BLOCK, row0 = (w.seq * a.c.kv_heads + w.head) * a.c.capacity;
                for (int u = w.u0; u < min(w.u0 + w.n, held) && ok; ++u, ++i) {
                    const int slot = i % P::RAWS;
                    if (i >= P::RAWS) ok = mbar_wait_bounded(&raw_empty[slot], (uint32_t)(i / P::RAWS - 1) & 1u, abort_flag);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&raw_full[slot], P::RAW);
                    tma_load_2d(raws + slot * P::RAW, &a.k_map, 0, row0 + u * BLOCK, &raw_full[slot]);
                    tma_load_2d(raws + slot * P::RAW + BLOCK * D, &a.v_map, 0, row0 + u * BLOCK, &raw_full[slot]);
                }
            } while (ok && w.next(a, deal));
        }
        __syncwarp();
    } else if (warp == 13) {
        if (elect_one()) {
            constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(BLOCK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);               // D f32, A and B f16
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);     // B: columns contiguous
            int i = 0, tile = 0, n[2] = {0, 0};          // units so far, tiles, units of a half
            bool ok = true;
            do {
                const int halves = min(PROMPT_ROWS, w.sp.n * deal.group - w.t * PROMPT_ROWS) > 128 ? 2 : 1;
                ok = mbar_wait_bounded(&q_full, (uint32_t)tile & 1u, abort_flag);
                tc::tc_fence_after();
                auto scores = [&](int x, int u) {
                    const int buffer = (n[x] + u) & 1;
                    const uint32_t q = smem_u32(qs + x * P::BOXES * P::QBOX), ks = smem_u32(units + (i + u) % P::UNITS * P::UNIT);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c)
                        tcw::mma_ss(tmem + x * P::HALF + buffer * BLOCK, row_desc(q + (c >> 2) * P::QBOX + (c & 3) * 32), row_desc(ks + (c >> 2) * P::KBOX + (c & 3) * 32),
                                    idesc_s, c == 0 ? 0u : 1u);
                    tc::tc_commit(&s_full[x][buffer]);
                };
                auto unit_there = [&](int u) {
                    ok = ok && mbar_wait_bounded(&unit_full[(i + u) % P::UNITS], (uint32_t)((i + u) / P::UNITS) & 1u, abort_flag);
                    tc::tc_fence_after();
                    return ok;
                };
                auto products = [&](int x, int u) {
                    const int mine = n[x] + u;
                    ok = ok && mbar_wait_bounded(&p_full[x][mine & 1], (uint32_t)(mine >> 1) & 1u, abort_flag);
                    if (!ok) return;
                    tc::tc_fence_after();
                    const uint32_t at = tmem + x * P::HALF, vs = smem_u32(units + (i + u) % P::UNITS * P::UNIT + P::BOXES * P::KBOX);
#pragma unroll
                    for (int c = 0; c < BLOCK / 16; ++c)
                        tc::tc_mma_ts(at + P::OUT, at + (mine & 1) * BLOCK + c * 8, value_desc(vs + c * 2048, P::KBOX), idesc_o, (u == 0 && c == 0) ? 0u : 1u);
                    tc::tc_commit(&o_done[x][mine & 1]);
                };
                if (ok && unit_there(0))
                    for (int x = 0; x < halves; ++x) scores(x, 0);
                for (int u = 0; u < w.n && ok; ++u) {
                    const bool next = u + 1 < w.n;
                    if (next && unit_there(u + 1)) scores(0, u + 1);
                    products(0, u);
                    if (halves > 1) {
                        if (next && ok) scores(1, u + 1);
                        products(1, u);
                    }
                    tc::tc_commit(&unit_empty[(i + u) % P::UNITS]);
                }
                i += w.n;
                for (int x = 0; x < halves; ++x) n[x] += w.n;
                ++tile;
            } while (ok && w.next(a, deal));
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ---- codes to FP16 ----
        const int me = tid - 256;
        int i = 0, r = 0;                                 // units, units of codes
        do {
            const int length = w.sp.pos + w.sp.n, held = length / BLOCK;
            const size_t at = (size_t)w.seq * a.c.kv_heads + w.head;
            if (i > 0)                                    // these warps are some units ahead: the tile's queries towards L2
                for (int j = me; j < min(PROMPT_ROWS, w.sp.n * deal.group - w.t * PROMPT_ROWS); j += 128) {
                    const int r = w.t * PROMPT_ROWS + j, token = r / deal.group;
                    const __half* q = a.q + (size_t)(w.sp.row + token) * a.ldq + (w.head * deal.group + r - token * deal.group) * D;
                    l2_prefetch(q);
                    if (D == 128) l2_prefetch(q + 64);
                }
            for (int u = w.u0; u < w.u0 + w.n; ++u, ++i) {
                const int slot = i % P::UNITS;
                if (i >= P::UNITS) tc::wait_uniform(&unit_empty[slot], (uint32_t)(i / P::UNITS - 1) & 1u, abort_flag);
                uint8_t* dst = units + slot * P::UNIT;
                auto put = [&](int side, int row, int chunk, const uint4& v) {           // 8 elements
                    *reinterpret_cast<uint4*>(dst + side * P::BOXES * P::KBOX + (chunk >> 3) * P::KBOX + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = v;
                };
                if (u < held) {
                    const int raw = r % P::RAWS;
                    tc::wait_uniform(&raw_full[raw], (uint32_t)(r / P::RAWS) & 1u, abort_flag);
                    const uint8_t* src = raws + raw * P::RAW;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        // chunk of four, row, keys or values, which four
                        const int item = j * 128 + me, chunk = (item >> 9) * 4 + (item & 3), side = (item >> 8) & 1, row = (item >> 2) & 63;
                        // eight lanes take rows r and r ^ 5
                        const int rr = (row & ~7) | ((row & 1) ? ((row & 7) >> 1) ^ 5 : (row & 7) >> 1);
                        const uint4 v = D == 128 ? *reinterpret_cast<const uint4*>(src + side * BLOCK * D + rr * 128 + ((chunk ^ (rr & 7)) << 4))
                                                 : *reinterpret_cast<const uint4*>(src + side * BLOCK * D + rr * 64 + ((chunk ^ ((rr >> 1) & 3)) << 4));
                        put(side, rr, 2 * chunk, make_uint4(codes_f16(v.x), codes_f16_hi(v.x), codes_f16(v.y), codes_f16_hi(v.y)));
                        put(side, rr, 2 * chunk + 1, make_uint4(codes_f16(v.z), codes_f16_hi(v.z), codes_f16(v.w), codes_f16_hi(v.w)));
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&raw_empty[raw]);
                    ++r;
                } else {
                    const int valid = length - u * BLOCK;
                    const __half* src[2] = {a.c.k_tail + (at * 2 + (u & 1)) * BLOCK * D, a.c.v_tail + (at * 2 + (u & 1)) * BLOCK * D};
                    for (int j = me; j < 2 * BLOCK * (D / 8); j += 128) {
                        const int chunk = j % (D / 8), row = j / (D / 8) % BLOCK, side = j / (D / 8) / BLOCK;
                        put(side, row, chunk, row < valid ? reinterpret_cast<const uint4*>(src[side] + row * D)[chunk] : make_uint4(0, 0, 0, 0));
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&unit_full[slot]);
            }
        } while (w.next(a, deal));
    } else {
        // ---- rows ----
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lane_tmem = tmem + x * P::HALF + ((uint32_t)((warp & 3) * 32) << 16), lane_o = lane_tmem + P::OUT;
        const float base = a.scale * LOG2E;
        const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.ldo * 2)) & 31) == 0;
        int n = 0, tile = -1;                             // units of this half; the tile's number
        // The queries of a tile to shared memory: that of the next one while the last products of this one run (its scores are all done).
        struct Mine { int all, r, token, head; bool live; } now;
        auto bring = [&](const Walk& w) {
            const int row0 = w.t * PROMPT_ROWS;
            Mine v;
            v.all = min(PROMPT_ROWS, w.sp.n * deal.group - row0);
            v.r = min(x * 128 + row, v.all - 1);
            v.token = (row0 + v.r) / deal.group;
            v.head = w.head * deal.group + (row0 + v.r) % deal.group;
            v.live = x * 128 + row < v.all;
            if (x * 128 < v.all) {
                // a warp's 32 rows, neighbouring lanes along a row; half of the loads at a time ahead of their stores
                constexpr int PER = D / 8, AT_ONCE = 32 / PER;
                const long long mine = (long long)(w.sp.row + v.token) * a.ldq + v.head * D;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint4 q[PER / 2];
#pragma unroll
                    for (int c = 0; c < PER / 2; ++c) {
                        const long long place = __shfl_sync(0xffffffffu, mine, (half * (PER / 2) + c) * AT_ONCE + lane / PER);
                        q[c] = __ldg(reinterpret_cast<const uint4*>(a.q + place) + lane % PER);
                    }
#pragma unroll
                    for (int c = 0; c < PER / 2; ++c) {
                        const int from = (warp & 3) * 32 + (half * (PER / 2) + c) * AT_ONCE + lane / PER, chunk = lane % PER;
                        const bool there = x * 128 + from < v.all;
                        *reinterpret_cast<uint4*>(qs + x * P::BOXES * P::QBOX + (chunk >> 3) * P::QBOX + from * 128 + (((chunk & 7) ^ (from & 7)) << 4)) =
                            there ? q[c] : make_uint4(0, 0, 0, 0);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
            return v;
        };
        now = bring(w);
        for (bool more = true; more;) {
            ++tile;
            const int row0 = w.t * PROMPT_ROWS;
            const size_t at = (size_t)w.seq * a.c.kv_heads + w.head;
            if (x * 128 >= now.all) {                     // not ahead of the others, whose arrivals would be taken for this half's
                tc::wait_uniform(&q_full, (uint32_t)tile & 1u, abort_flag);
                if (lane == 0) s_without[warp] += w.n;
                __syncwarp();
                more = w.next(a, deal);
                if (more) now = bring(w);
                continue;
            }
            const int held = (w.sp.pos + w.sp.n) / BLOCK, p = w.sp.pos + now.token;
            const int first = w.sp.pos + row0 / deal.group, last = w.sp.pos + (row0 + now.all - 1) / deal.group;   // positions of the tile
            const float* k_scale = a.c.k_scale + at * (a.c.capacity / BLOCK);
            const float* v_scale = a.c.v_scale + at * (a.c.capacity / BLOCK);
            float ks = w.u0 < held ? k_scale[w.u0] : 1.0f, vs = w.u0 < held ? v_scale[w.u0] : 1.0f;
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < w.n; ++j, ++n) {
                const int u = w.u0 + j;
                const float factor = base * ks;
                float inv = power_of_two(-exponent_of(vs)), ev = (float)exponent_of(vs);
                if (j + 1 < w.n) { ks = u + 1 < held ? k_scale[u + 1] : 1.0f; vs = u + 1 < held ? v_scale[u + 1] : 1.0f; }
                const uint32_t scores = lane_tmem + (n & 1) * BLOCK;
                tc::wait_uniform(&s_full[x][n & 1], (uint32_t)(n >> 1) & 1u, abort_flag);
                tc::tc_fence_after();
                if (ev == 0.0f) {                         // a scale of one, which a block of zeros has too
                    const int i = n + s_without[warp], slot = i % P::UNITS;
                    if (no_values(reinterpret_cast<const uint4*>(units + slot * P::UNIT + P::BOXES * P::KBOX), BLOCK * D / 8, &unit_full[slot], (uint32_t)(i / P::UNITS) & 1u, abort_flag)) {
                        ev = (float)NO_VALUES;
                        inv = power_of_two(-NO_VALUES);
                    }
                }
                uint32_t s[4][16];
#pragma unroll
                for (int c = 0; c < 4; ++c) tc::tmem_ld<16>(scores + c * 16, s[c]);
                tc::tmem_wait_ld();
                const int lim = p - u * BLOCK;            // the last key of the unit that the row sees
                if ((u + 1) * BLOCK - 1 > first) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (c * 16 + e > lim) s[c][e] = __float_as_uint(-INFINITY);
                }
                if (last - u * BLOCK >= a.window) {
                    const int low = lim - a.window;       // the last key that is too far behind
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (c * 16 + e <= low) s[c][e] = __float_as_uint(-INFINITY);
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int e = 1; e < 16; ++e) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][e]));
                }
                const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), factor, ev);
                float before = 1.0f;
                const bool moved = top > m + MOST_TOP;
                if (moved) {
                    before = ex2(m - (top - LEAST_TOP));
                    m = top - LEAST_TOP;
                    l *= before;
                }
                const float shift = ev - (m == -INFINITY ? 0.0f : m);
                const float2 factor2 = make_float2(factor, factor), shift2 = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t f[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint32_t* pair = &s[2 * c + (e >> 3)][2 * e & 15];
                        float2 y = fma2(make_float2(__uint_as_float(pair[0]), __uint_as_float(pair[1])), factor2, shift2);
                        y.x = ex2(y.x);
                        y.y = ex2(y.y);
                        sum[e & 1] = add2(sum[e & 1], y);
                        f[e] = pack_f16(y.x, y.y);
                    }
                    tc::tmem_st16(scores + c * 16, f);
                }
                sum[0] = add2(sum[0], sum[1]);
                l = fmaf(sum[0].x + sum[0].y, inv, l);
                // A barrier for even and one for odd products: a parity does not tell a phase from the one after the next, and these scores came
                // behind the products of the unit before the last.
                if (j > 0 && __any_sync(0xffffffffu, moved)) {
                    tc::wait_uniform(&o_done[x][(n - 1) & 1], (uint32_t)((n - 1) >> 1) & 1u, abort_flag);
                    tc::tc_fence_after();
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tc::tmem_ld<16>(lane_o + c, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * before);
                        tc::tmem_st16(lane_o + c, o);
                    }
                }
                tc::tmem_wait_st();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[x][n & 1]);     // one for even and one for odd units: a warp may be a unit ahead of another
            }
            const bool alone = w.begins && w.ends, live = now.live;
            const int r = now.r;
            float* part = a.partial + (2 * (size_t)blockIdx.x + (w.begins ? 1 : 0)) * partial_floats(PROMPT_ROWS, D);
            __half* out = a.out + (size_t)(w.sp.row + now.token) * a.ldo + now.head * D;
            more = w.next(a, deal);
            if (more) now = bring(w);
            else if (tid == 0) leave_word(a, deal, w, start);
            tc::wait_uniform(&o_done[x][(n - 1) & 1], (uint32_t)((n - 1) >> 1) & 1u, abort_flag);
            tc::tc_fence_after();
            const bool ok = *abort_flag == 0;
            const float inv_l = 1.0f / l;
            for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tc::tmem_ld<16>(lane_o + c, o);
                tc::tmem_wait_ld();
                if (!live || !ok) continue;
                if (alone) {
                    uint32_t h[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[e] = pack_f16(__uint_as_float(o[2 * e]) * inv_l, __uint_as_float(o[2 * e + 1]) * inv_l);
                    if (wide) {                           // a sector at once
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + c), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]), "r"(h[4]),
                                     "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(out + c);
                        dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
                        dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) reinterpret_cast<uint4*>(part)[(c + e) / 4 * PROMPT_ROWS + r] = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (live && ok && !alone) { part[PROMPT_ROWS * D + r] = m; part[PROMPT_ROWS * (D + 1) + r] = l; }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, P::TMEM);
    }
}

}  // namespace cache8
}  // namespace twm
