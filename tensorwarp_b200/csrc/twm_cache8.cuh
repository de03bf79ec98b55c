// twm_cache8.cuh — the key/value cache held in 8 bits (include/twm_serve.h): its layout, and the append of new tokens.
#pragma once

#include <cuda_fp8.h>

#include "../../include/twm_serve.h"
#include "twm_common.cuh"

namespace twm {
namespace cache8 {

constexpr int BLOCK = TWM_CACHE8_BLOCK;

struct Cache {
    int seqs, kv_heads, capacity;
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    __half *k_tail, *v_tail;
};

// The rows of a call (host pointers of the caller's device arrays).
struct Rows {
    const int* row_start;        // [seqs + 1] or null: one row a sequence
    const int* start;            // [seqs]
    int rows, max_rows;
};

// One sequence's share of a call: its first row, position and number of rows, cut to what the call and the cache hold, whatever
// the arrays say.
struct Span { int row, pos, n; };
__device__ __forceinline__ Span span_of(const Rows& r, int seq, int capacity)
{
    Span s;
    s.pos = r.start[seq];
    int end;
    if (r.row_start != nullptr) {
        s.row = min(max(r.row_start[seq], 0), r.rows);
        end = min(max(r.row_start[seq + 1], s.row), r.rows);
    } else {
        s.row = seq;
        end = seq + 1;
    }
    s.n = min(end - s.row, r.max_rows);
    s.n = s.pos < 0 ? 0 : min(s.n, capacity - min(s.pos, capacity));
    return s;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8])
{
    uint4 o;
    uint32_t* w = &o.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return o;
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8])
{
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// The exponent e of a block's scale 2^e: the smallest with amax <= 448 * 2^e = 1.75 * 2^(8 + e).  amax is a finite FP16 value.
__device__ __forceinline__ int scale_exponent(float amax)
{
    if (!(amax > 0.0f)) return 0;
    const uint32_t bits = __float_as_uint(amax);
    return (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Whether a number has no place in the cache as FP16; it becomes NaN (a key's) or zero (a value's).
__device__ __forceinline__ bool not_finite(float& x, int side)
{
    if (fabsf(x) < 65520.0f) return false;       // what rounds to at most 65504
    x = side == 0 ? NAN : 0.0f;
    return true;
}

struct AppendArgs {
    Cache c;
    Rows r;
    __half* q_out;
    const __half* qkv;
    const float *bias, *rope;
    long ldq, ldqkv;
    int num_heads;
    int apart;                   // 1: every query head has CTAs of its own
};

// CTA = (64-token block of positions, key/value head, sequence): rotates the queries of the head's group and the keys of its new
// tokens, and brings keys and values into the cache.  A block that is full now is put together in shared memory (its earlier tokens
// from the tail) for the largest value, then rounded; the two newest blocks go to the tail.  A call may begin inside a block whose
// earlier tokens are read from a half of the tail that the call's last block takes over: both are then the work of the CTA of the
// first block, in that order.  Of a token or a few every thread has one item, so that all loads are on their way at once.  Prompts are
// bound by memory and take a CTA for every query head of a block as well (4000 tokens, 28 heads: 29 us without, 23 us with), from a quarter of a block
// on: there it gains for few sequences and costs for many, which from half a block on gain too (40 heads on 8, us without and with: 8 rows of 1, 8 and
// 64 sequences 4.9 and 3.6, 5.1 and 4.3, 10.2 and 14.6; 16 rows 5.7 and 3.8, 5.9 and 4.7, 13.2 and 16.2; 32 rows 7.4 and 4.1, 7.6 and 5.1, 24.3 and 23.7).
constexpr int APPEND_THREADS = 256;
template <int D>
__global__ void __launch_bounds__(APPEND_THREADS)
append_kernel(const __grid_constant__ AppendArgs a)
{
    constexpr int OCTS = D / 16;                 // runs of 8 pairs of a head
    __shared__ __align__(16) __half tile[2][BLOCK][D];          // keys, values
    __shared__ float amax[2][APPEND_THREADS / 32];
    __shared__ int odd[BLOCK];                                  // tokens whose value is no number
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int seq = blockIdx.z, h = blockIdx.y % a.c.kv_heads, tid = threadIdx.x;
    const Span sp = span_of(a.r, seq, a.c.capacity);
    const int first = sp.pos / BLOCK, end = sp.pos + sp.n;
    const int mine = first + blockIdx.x;
    if (sp.n <= 0 || mine * BLOCK >= end) return;
    const int group = a.num_heads / a.c.kv_heads, kv_dim = a.c.kv_heads * D, q_dim = a.num_heads * D;
    const int last = (end - 1) / BLOCK;
    const bool inside = sp.pos % BLOCK != 0;     // the first block's earlier tokens come from the tail

    // one run of 8 pairs: elements col ... and col + D/2 ... of a row, with bias, turned by position `pos` or not
    auto load_pairs = [&](int pos, int col, int oct, bool turn, float (&lo)[8], float (&hi)[8]) {
        const __half* src = a.qkv + (size_t)(sp.row + pos - sp.pos) * a.ldqkv + col + oct * 8;
        unpack8(*reinterpret_cast<const uint4*>(src), lo);
        unpack8(*reinterpret_cast<const uint4*>(src + D / 2), hi);
        if (a.bias != nullptr) {
            float b[8];
            load8(a.bias + col + oct * 8, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[i] += b[i];
            load8(a.bias + col + oct * 8 + D / 2, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) hi[i] += b[i];
        }
        if (turn && a.rope != nullptr) {
            float c[8], s[8];
            load8(a.rope + (size_t)pos * D + oct * 8, c);
            load8(a.rope + (size_t)pos * D + D / 2 + oct * 8, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) {        // not contracted: the plain product and sum, whoever rotates
                const float x = lo[i], y = hi[i];
                lo[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
                hi[i] = __fadd_rn(__fmul_rn(x, s[i]), __fmul_rn(y, c[i]));
            }
        }
    };

    const int p0 = max(sp.pos, mine * BLOCK), p1 = min(end, (mine + 1) * BLOCK);
    auto store_query = [&](int pos, int head, int oct, const float (&lo)[8], const float (&hi)[8]) {
        __half* dst = a.q_out + (size_t)(sp.row + pos - sp.pos) * a.ldq + head * D + oct * 8;
        *reinterpret_cast<uint4*>(dst) = pack8(lo);
        *reinterpret_cast<uint4*>(dst + D / 2) = pack8(hi);
    };
    if (a.apart && blockIdx.y >= a.c.kv_heads) {
        const int head = blockIdx.y - a.c.kv_heads;
#pragma unroll 2
        for (int i = tid; i < (p1 - p0) * OCTS; i += APPEND_THREADS) {
            float lo[8], hi[8];
            load_pairs(p0 + i / OCTS, head * D, i % OCTS, true, lo, hi);
            store_query(p0 + i / OCTS, head, i % OCTS, lo, hi);
        }
        return;
    }

    const size_t at = (size_t)seq * a.c.kv_heads + h;
    __half* tails[2] = {a.c.k_tail + at * 2 * BLOCK * D, a.c.v_tail + at * 2 * BLOCK * D};
    // a key's (side 0) or value's run of 8 pairs into the block's tile and its half of the tail
    auto put = [&](int side, int b, int pos, int oct, const float (&lo)[8], const float (&hi)[8], bool to_tail, bool to_codes) {
        const uint4 l = pack8(lo), u = pack8(hi);
        if (to_codes) {
            *reinterpret_cast<uint4*>(&tile[side][pos % BLOCK][oct * 8]) = l;
            *reinterpret_cast<uint4*>(&tile[side][pos % BLOCK][oct * 8 + D / 2]) = u;
        }
        if (to_tail) {
            __half* dst = tails[side] + ((b & 1) * BLOCK + pos % BLOCK) * D + oct * 8;
            *reinterpret_cast<uint4*>(dst) = l;
            *reinterpret_cast<uint4*>(dst + D / 2) = u;
        }
    };
    auto odd_ones = [&](float (&lo)[8], float (&hi)[8], int side) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) any |= not_finite(lo[j], side) | not_finite(hi[j], side);
        return any;
    };
    auto keep = [&](int b, bool to_tail, bool to_codes) {
        const int b0 = max(sp.pos, b * BLOCK), b1 = min(end, (b + 1) * BLOCK), tokens = b1 - b0;
        if (tid < BLOCK) odd[tid] = 0;
        __syncthreads();
        if (!a.apart && b == mine && tokens * (group + 2) * OCTS <= APPEND_THREADS) {        // an item a thread: queries, keys, values
            const int oct = tid % OCTS, kind = tid / OCTS % (group + 2), pos = b0 + tid / (OCTS * (group + 2));
            const bool there = pos < b1;
            float lo[8], hi[8];
            if (there) {
                load_pairs(pos, kind < group ? (h * group + kind) * D : q_dim + (kind - group) * kv_dim + h * D, oct, kind <= group, lo, hi);
                if (kind < group) store_query(pos, h * group + kind, oct, lo, hi);
                else if (odd_ones(lo, hi, kind - group) && kind > group) odd[pos % BLOCK] = 1;
            }
            __syncthreads();
            if (there && kind >= group) {
                if (kind == group && oct == 0 && odd[pos % BLOCK]) lo[0] = NAN;
                put(kind - group, b, pos, oct, lo, hi, to_tail, to_codes);
            }
        } else {
            if (!a.apart && b == mine)
                for (int i = tid; i < tokens * group * OCTS; i += APPEND_THREADS) {
                    const int oct = i % OCTS, head = h * group + i / OCTS % group, pos = b0 + i / (OCTS * group);
                    float lo[8], hi[8];
                    load_pairs(pos, head * D, oct, true, lo, hi);
                    store_query(pos, head, oct, lo, hi);
                }
            // values, then keys, which may have to say that the value is none
#pragma unroll 1
            for (int side = 1; side >= 0; --side) {
#pragma unroll 2
                for (int i = tid; i < tokens * OCTS; i += APPEND_THREADS) {
                    const int oct = i % OCTS, pos = b0 + i / OCTS;
                    float lo[8], hi[8];
                    load_pairs(pos, q_dim + side * kv_dim + h * D, oct, side == 0, lo, hi);
                    const bool any = odd_ones(lo, hi, side);
                    if (side == 1 && any) odd[pos % BLOCK] = 1;
                    if (side == 0 && oct == 0 && odd[pos % BLOCK]) lo[0] = NAN;
                    put(side, b, pos, oct, lo, hi, to_tail, to_codes);
                }
                __syncthreads();
            }
        }
        if (!to_codes) return;
        for (int i = tid; i < 2 * (b0 - b * BLOCK) * (D / 8); i += APPEND_THREADS) {        // the block's earlier tokens
            const int piece = i % (D / 8), side = i / (D / 8) % 2, row = i / (2 * (D / 8));
            *reinterpret_cast<uint4*>(&tile[side][row][piece * 8]) =
                *reinterpret_cast<const uint4*>(tails[side] + ((b & 1) * BLOCK + row) * D + piece * 8);
        }
        __syncthreads();
        // half of the threads take the keys, half the values
        const int side = tid / (APPEND_THREADS / 2), t = tid % (APPEND_THREADS / 2);
        constexpr int PIECES = BLOCK * D / 8;
        const uint4* src = reinterpret_cast<const uint4*>(&tile[side][0][0]);
        float m = 0.0f;
        for (int i = t; i < PIECES; i += APPEND_THREADS / 2) {
            float f[8];
            unpack8(src[i], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(f[j]));          // NaN: m
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((tid & 31) == 0) amax[side][t / 32] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < APPEND_THREADS / 64; ++w) m = fmaxf(m, amax[side][w]);
        const int e = scale_exponent(m);
        const float inv = power_of_two(-e);
        uint8_t* codes = (side ? a.c.v : a.c.k) + (at * a.c.capacity + (size_t)b * BLOCK) * D;
        for (int i = t; i < PIECES; i += APPEND_THREADS / 2) {
            float f[8];
            unpack8(src[i], f);
            uint32_t w[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * j] * inv, f[2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                w[j >> 1] = (j & 1) ? (w[j >> 1] | (c << 16)) : c;
            }
            *reinterpret_cast<uint2*>(codes + (size_t)i * 8) = make_uint2(w[0], w[1]);
        }
        if (t == 0) (side ? a.c.v_scale : a.c.k_scale)[at * (a.c.capacity / BLOCK) + b] = power_of_two(e);
    };
    // block `late` takes over the half of the tail that the first block still reads
    const int late = inside && last - first >= 2 ? last - ((last - first) & 1) : -1;
    const bool full = (mine + 1) * BLOCK <= end;
    keep(mine, mine >= last - 1 && mine != late, full);
    if (mine == first && late >= 0) {
        __syncthreads();
        keep(late, true, false);
    }
}

}  // namespace cache8
}  // namespace twm
