// twm_cache8_attn.cuh — softmax attention over the cache held in 8 bits: how the work is dealt out, attention of few rows a sequence, and
// the merge of what several CTAs have of a tile.
//
// Mathematics, common to all kernels.  Keys are c_k 2^ek and values c_v 2^ev with one ek and ev a block of 64 tokens (0 in the tail, whose
// tokens are FP16).  The codes enter the tensor core as FP16, exactly.  The exponent of key j for a row is
//     x_j = (q . c_k) (scale 2^ek log2 e) + ev,
// so that 2^x_j is the factor of the CODES c_v in the output, and 2^(x_j - ev) the weight that belongs into the sum of weights:
//     o = sum 2^(x_j - m) c_v / sum 2^(x_j - m) 2^-ev.
// One fused multiply-add an element as without scales.  The running reference m is that of x_j, scale of the value included: it is set
// so that the largest factor is 2^7 and moves only when one would pass 2^15.  So a row's largest factor so far lies between them, whatever the scales of
// its blocks are, and a factor is rounded to FP16 by 2^-11 of itself down to 2^-14, and by at most 2^-32 of the largest one below: the values' codes
// have four bits, and sums, scores and statistics are FP32.
// For that ev has to say how large values are.  A block of zeros has scale 1: its ev is NO_VALUES, below all others, so that it weighs in the sum and
// leaves the reference to the others.  The tail has ev 0 however small its values are, but comes last: no factor of codes is taken behind it.
#pragma once

#include "twm_cache8.cuh"
#include "twm_gemm_tc.cuh"

namespace twm {
namespace cache8 {

constexpr float LOG2E = 1.4426950408889634f;

struct __align__(16) Join {
    int parts;                   // CTAs that have keys of it; 0: no such tile
    int rows, row0;              // rows of the tile, and the first of them among those of its sequence and head
    int head, row;               // key/value head, and the sequence's first row in the call
    int unused[3];
};
struct AttnArgs {
    Cache c;
    Rows r;
    __half* out;
    const __half* q;
    long ldo, ldq;
    int num_heads, window;       // window: INT_MAX = all
    float scale;
    struct Join* joins;          // [CTAs]: the tile that a CTA began and did not end
    float* partial;              // [2 CTAs][tile]: what a CTA has of its first and of its last tile, where others have the rest
    alignas(64) CUtensorMap k_map, v_map;        // bytes [cached rows][D], boxes of a block, swizzled
};

// ------------------------------------------------------------------------------------------------------ dealing out --
// The rows of a sequence and key/value head, i * group + (head in the group), are cut into tiles of `tile` rows; the keys that any row
// of a tile sees into units of 64 tokens, blocks of the cache.  All units of a call stand in one line, by sequence, head, tile
// and key, and every CTA takes an equal run of it, whatever the lengths: a CTA's first and last tile may be shared with its neighbours, which
// merge_kernel then joins; the ones between are its own.
struct Tile { int lo, end; };    // first unit, unit behind the last
__device__ __forceinline__ Tile tile_units(const Span& sp, int t, int tile, int group, int window)
{
    const int rows = sp.n * group;
    int first = sp.pos, last = sp.pos + sp.n - 1;
    if (rows > tile) {
        first = sp.pos + t * tile / group;
        last = sp.pos + (min(rows, (t + 1) * tile) - 1) / group;
    }
    return {(window > first ? 0 : first - window + 1) / BLOCK, last / BLOCK + 1};
}
// A tile also takes time of its own, `extra` units' worth, which stand ahead of its units in the line.
struct Deal {
    int group, tile, window, extra;
    int least;                   // units of a CTA at least
    __device__ __forceinline__ int tiles(const Span& sp) const { return sp.n * group <= tile ? 1 : (sp.n * group + tile - 1) / tile; }
    __device__ __forceinline__ int units(const Span& sp, int t) const
    {
        const Tile x = tile_units(sp, t, tile, group, window);
        return extra + x.end - x.lo;
    }
    // units of one head of a sequence, by all lanes of a warp
    __device__ __forceinline__ long long units_by_warp(const Span& sp) const
    {
        const int n = sp.n > 0 ? tiles(sp) : 0;
        long long u = 0;
        for (int t = threadIdx.x & 31; t < n; t += 32) u += units(sp, t);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
        return u;
    }
};

// x / y, neither negative; a 64-bit division takes several times as long as a 32-bit one
__device__ __forceinline__ long long quotient(long long x, long long y) { return ((x | y) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)y) : x / y; }

// Where a CTA's run begins, found by the whole CTA.
struct Start {
    bool out;                    // whether a sequence is out of the call
    long long units;             // of the CTA
    long long share;             // of every CTA but the last ones
    long long before;            // units of the sequence ahead of the run
    int seq;
};
// A thread takes neighbouring sequences; where a sequence can have several tiles, a warp does, its lanes the tiles.
template <int THREADS>
__device__ __forceinline__ Start find_start(const AttnArgs& a, const Deal& deal, int cta, int ctas)
{
    __shared__ long long sums[THREADS / 32];
    __shared__ Start found;
    const int tid = threadIdx.x, lane = tid & 31;
    const bool by_warp = (long long)a.r.max_rows * deal.group > deal.tile;
    const int takers = by_warp ? THREADS / 32 : THREADS, me = by_warp ? tid / 32 : tid;
    const int per = (a.c.seqs + takers - 1) / takers, s0 = min(a.c.seqs, me * per), s1 = min(a.c.seqs, s0 + per);
    auto units = [&](int s) {
        const Span sp = span_of(a.r, s, a.c.capacity);
        return (by_warp ? deal.units_by_warp(sp) : sp.n > 0 ? (long long)deal.units(sp, 0) : 0LL) * a.c.kv_heads;
    };
    long long mine = 0;
    bool out = false;
    for (int s = s0; s < s1; ++s) {
        mine += units(s);
        out |= a.r.start[s] < 0;
    }
    long long upto = mine;
    if (!by_warp) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
    }
    if (lane == 31) sums[tid / 32] = upto;
    if (tid == 0) found = {false, 0, 0, 0, 0};
    out = __syncthreads_or(out);
    long long base = 0, total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < tid / 32) base += sums[w];
        total += sums[w];
    }
    upto += base;
    const long long share = max((long long)deal.least, quotient(total + ctas - 1, ctas)), begin = min(total, share * cta), end = min(total, begin + share);
    if (begin < end && upto - mine <= begin && begin < upto) {           // the same in all lanes of a warp where warps take sequences
        long long at = upto - mine;
        for (int s = s0; s < s1; ++s) {
            const long long n = units(s);
            if (begin < at + n) {
                if (!by_warp || lane == 0) found = {false, end - begin, share, begin - at, s};
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    Start start = found;
    start.out = out;
    return start;
}

// The tiles of a CTA's run, one after another.
struct Walk {
    long long left;              // of the run, behind the current tile
    int seq, head, t;            // the current tile
    int u0, n;                   // its first unit and number of units in this run; none at all where the run ends with a tile's extra
    bool begins, ends;           // whether the run has the tile's first and last unit
    Span sp;
    Tile whole;

    __device__ __forceinline__ void take(const Deal& d, int skip)
    {
        whole = tile_units(sp, t, d.tile, d.group, d.window);
        const int all = d.extra + whole.end - whole.lo, to = (int)min((long long)all, skip + left), from = max(skip - d.extra, 0);
        u0 = whole.lo + from;
        n = max(to - d.extra, 0) - from;
        begins = from == 0;
        ends = to == all;
        left -= to - skip;
    }
    // by all lanes of a warp; false where the run has no unit
    __device__ __forceinline__ bool begin(const AttnArgs& a, const Deal& d, const Start& s)
    {
        if (s.units == 0) return false;
        left = s.units;
        seq = s.seq;
        sp = span_of(a.r, seq, a.c.capacity);
        const int tiles = d.tiles(sp), lane = threadIdx.x & 31;
        const long long per = tiles == 1 ? d.units(sp, 0) : d.units_by_warp(sp);
        head = (int)quotient(s.before, per);
        long long rest = s.before - head * per;                          // 32 tiles' units fit 32 bits (cached rows / 64 each), a head's need not
        t = 0;
        while (tiles > 1) {                                              // 32 tiles at a time
            const int mine = t + lane < tiles ? d.units(sp, t + lane) : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned int in = __ballot_sync(0xffffffffu, rest < upto);
            if (in != 0) {
                const int x = __ffs(in) - 1;
                rest -= __shfl_sync(0xffffffffu, upto - mine, x);
                t += x;
                break;
            }
            rest -= __shfl_sync(0xffffffffu, upto, 31);
            t += 32;
        }
        take(d, (int)rest);
        return n > 0;
    }
    __device__ __forceinline__ bool next(const AttnArgs& a, const Deal& d)
    {
        if (left <= 0) return false;
        if (++t >= d.tiles(sp)) {
            t = 0;
            if (++head >= a.c.kv_heads) {
                head = 0;
                do sp = span_of(a.r, ++seq, a.c.capacity); while (sp.n <= 0);
            }
        }
        take(d, 0);
        return n > 0;            // a run that ends with a tile's extra ends ahead of it
    }
};

// The same where every sequence has one tile and there are at most 128 of them: every warp finds the start by itself, a few neighbouring sequences
// a lane, in 32 bits (units of all sequences: cached rows / 64, and a tile's extra each).  2.3 + 1.0 thousand clocks of a call for one sequence
// with find_start and begin, 1.5 + 0.15 thousand this way.
constexpr int START_BY_WARP = 128;
__device__ __forceinline__ bool begin_by_warp(const AttnArgs& a, const Deal& d, int cta, int ctas, Start& start, Walk& w)
{
    const int lane = threadIdx.x & 31, per = (a.c.seqs + 31) / 32, s0 = min(a.c.seqs, lane * per), s1 = min(a.c.seqs, s0 + per);
    int mine = 0;
    bool out = false;
    for (int s = s0; s < s1; ++s) {
        const Span sp = span_of(a.r, s, a.c.capacity);
        if (sp.n > 0) mine += d.units(sp, 0) * a.c.kv_heads;
        out |= sp.pos < 0;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31), share = max(d.least, (total + ctas - 1) / ctas);
    const int begin = (int)min((long long)share * cta, (long long)total), end = min(total, begin + share);
    start = {__any_sync(0xffffffffu, out) != 0, end - begin, share, 0, 0};
    if (begin >= end) return false;
    const unsigned int in = __ballot_sync(0xffffffffu, begin < upto);
    const int owner = __ffs(in) - 1;
    int before = begin - __shfl_sync(0xffffffffu, upto - mine, owner), seq = owner * per, units = 0;
    for (;; ++seq) {                                                     // every lane along the owner's sequences
        w.sp = span_of(a.r, seq, a.c.capacity);
        units = w.sp.n > 0 ? d.units(w.sp, 0) : 0;
        if (before < units * a.c.kv_heads) break;
        before -= units * a.c.kv_heads;
    }
    w.left = end - begin;
    w.seq = seq;
    w.head = before / units;
    w.t = 0;
    w.take(d, before - w.head * units);
    return w.n > 0;
}

// Leaves word for merge_kernel of the run's last tile (`w` stands there), or that there is none.
__device__ __forceinline__ void leave_word(const AttnArgs& a, const Deal& d, const Walk& w, const Start& s)
{
    const int row0 = w.t * d.tile;
    const bool open = w.n > 0 && w.begins && !w.ends;
    a.joins[blockIdx.x] = {open ? 1 + (int)((w.whole.end - w.u0 - w.n + s.share - 1) / s.share) : 0, min(d.tile, w.sp.n * d.group - row0), row0, w.head, w.sp.row, {0, 0, 0}};
}

// Rows of sequences that are out of the call are zeros; CTA `cta` of `ctas` takes its share of the sequences.
__device__ __forceinline__ void zero_rows(const AttnArgs& a, int D, int cta, int ctas, int tid, int threads)
{
    for (int s = cta; s < a.c.seqs; s += ctas) {
        if (a.r.start[s] >= 0) continue;
        const int r0 = a.r.row_start ? min(max(a.r.row_start[s], 0), a.r.rows) : s;
        const int r1 = a.r.row_start ? min(min(max(a.r.row_start[s + 1], r0), a.r.rows), r0 + a.r.max_rows) : s + 1;
        const int pieces = a.num_heads * D / 8;
        for (long long i = tid; i < (long long)(r1 - r0) * pieces; i += threads)
            *reinterpret_cast<uint4*>(a.out + (r0 + i / pieces) * a.ldo + i % pieces * 8) = make_uint4(0, 0, 0, 0);
    }
}

// A tile in the workspace: [tile rows][D] sums, then the rows' references and sums of weights.
__host__ __device__ inline size_t partial_floats(int tile, int D) { return (size_t)tile * (D + 2); }

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// the exponent of a block's scale, from the scale
__device__ __forceinline__ int exponent_of(float scale) { return (int)(__float_as_uint(scale) >> 23) - 127; }

constexpr float LEAST_TOP = 7.0f, MOST_TOP = 15.0f;                      // logarithms between which a row's largest factor lies
constexpr int NO_VALUES = -64;

// --------------------------------------------------------------------------------------------- few rows a sequence --
// Up to 8 NT rows a sequence and key/value head (the query heads that share it, times the new tokens): they are one tile, and every key is
// read once.  Bound by HBM (96 sequences of up to 6000 tokens, 40 heads on 8: 119 us, 6.18 TB/s).  Four consumer warps take 16 keys each of a
// unit; a producer warp brings units by TMA into a ring that runs on over the borders of tiles, the tail's FP16 rows among them (keys and
// values in a stage each).  S^T = K Q^T and O^T += V^T P^T as mma.m16n8k16 with the keys, and then the head's elements, as the 16 rows, so that eight
// rows of queries are a whole operand (with NT = 2 and D = 128 registers do not reach: 434 bytes of them are stored, and 96 sequences of 4000 tokens, 40
// heads on 8, take 257 us with two new tokens each, 125 with one).  Elements and keys may stand in any order in a sum: lane (g, t) takes D / 4 elements of keys g and g + 8 for
// the scores (4 codes a k-step of both registers), and D / 8 elements of four keys for the output, whose codes are paired by a byte permutation; at
// D = 128 both reads are free of bank conflicts in the layout that the TMA's swizzle leaves.  P^T needs only a transposition of 8 x 8.  Each warp has
// its own m; when the tile ends the four add up in shared memory, while the next tile's queries are on their way.
constexpr int FEW_EXTRA = 4;                                             // a tile's own time, in units (96 sequences: 1 124.5 us, 2 121.9, 4 120.8)
constexpr int FEW_LEAST = 1;                                             // units of a CTA at least (2049 tokens, 28 heads: 1 9.2 us, 2 9.5, 4 10.4)
constexpr int FEW_WARPS = 4, FEW_THREADS = 32 * FEW_WARPS + 32;
template <int D, int NT>
struct Few {
    static constexpr int STAGE = 2 * BLOCK * D;                          // bytes: codes of keys and values, or the tail's of one of them
    static constexpr int CTAS = D == 64 && NT == 1 ? 3 : 2;              // to an SM, as registers allow (D = 64, 40 sequences: two 22.7 us, three 20.8)
    static constexpr int STAGES = CTAS == 3 ? 6 : (NT == 1 ? 5 : 4) * 128 / D;
    static constexpr int TILE = 8 * NT;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + (size_t)FEW_WARPS * TILE * D * 4;
};

__device__ __forceinline__ uint32_t codes_f16(uint32_t pair)            // two codes in the low half
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(pair));
    return r;
}
__device__ __forceinline__ uint32_t codes_f16_hi(uint32_t pair)         // in the high half
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(pair));
    return r;
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D, int NT>
__global__ void __launch_bounds__(FEW_THREADS, Few<D, NT>::CTAS)
few_kernel(const __grid_constant__ AttnArgs a)
{
    using F = Few<D, NT>;
    constexpr int KS = D / 16, WK = D / 64, DPL = D / 8;     // k-steps, 16-byte words a key and lane for the scores, elements of a lane for the output
    extern __shared__ uint8_t few_raw[];
    __shared__ uint64_t full[F::STAGES], empty[F::STAGES];
    __shared__ float s_m[FEW_WARPS][F::TILE], s_l[FEW_WARPS][F::TILE];
    __shared__ int s_abort;
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_raw) + 1023) & ~(uintptr_t)1023);
    float4* join = reinterpret_cast<float4*>(stages + (size_t)F::STAGES * F::STAGE);         // [warp][row][D / 4], a row's turned about by the row
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < F::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], FEW_WARPS); }
        s_abort = 0;
        mbar_fence_init();
    } else if (tid == 32 * FEW_WARPS) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.k_map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.v_map)) : "memory");
    }
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const Deal deal = {a.num_heads / a.c.kv_heads, F::TILE, a.window, FEW_EXTRA, FEW_LEAST};
    Start start;
    Walk w;
    bool any;
    if (a.c.seqs <= START_BY_WARP) {
        any = begin_by_warp(a, deal, blockIdx.x, gridDim.x, start, w);
        __syncthreads();                                                 // the barriers are there
    } else {
        start = find_start<FEW_THREADS>(a, deal, blockIdx.x, gridDim.x);
        any = w.begin(a, deal, start);
    }
    if (start.out) zero_rows(a, D, blockIdx.x, gridDim.x, tid, FEW_THREADS);
    if (!any) {
        if (tid == 0) a.joins[blockIdx.x].parts = 0;
        return;
    }
    volatile int* abort_flag = &s_abort;

    if (warp == FEW_WARPS) {
        if (lane == 0) {
            int i = 0;
            bool ok = true;
            auto slot = [&]() {                                          // the next stage, free
                const int x = i % F::STAGES;
                if (i >= F::STAGES) ok = ok && mbar_wait_bounded(&empty[x], (uint32_t)(i / F::STAGES - 1) & 1u, abort_flag);
                ++i;
                return x;
            };
            do {
                const int length = w.sp.pos + w.sp.n, held = length / BLOCK;         // units that are codes
                const size_t at = (size_t)w.seq * a.c.kv_heads + w.head;
                const int row0 = (w.seq * a.c.kv_heads + w.head) * a.c.capacity;
                for (int u = w.u0; u < w.u0 + w.n && ok; ++u) {
                    if (u < held) {
                        const int x = slot();
                        if (!ok) break;
                        mbar_arrive_expect_tx(&full[x], F::STAGE);
                        tma_load_2d(stages + x * F::STAGE, &a.k_map, 0, row0 + u * BLOCK, &full[x]);
                        tma_load_2d(stages + x * F::STAGE + BLOCK * D, &a.v_map, 0, row0 + u * BLOCK, &full[x]);
                    } else {                                             // the tokens of the tail that are there
                        const uint32_t bytes = (uint32_t)(length - u * BLOCK) * D * 2;
                        const size_t from = (at * 2 + (u & 1)) * BLOCK * D;
                        for (int side = 0; side < 2; ++side) {
                            const int x = slot();
                            if (!ok) break;
                            mbar_arrive_expect_tx(&full[x], bytes);
                            bulk_g2s(stages + x * F::STAGE, (side ? a.c.v_tail : a.c.k_tail) + from, bytes, &full[x]);
                        }
                    }
                }
            } while (ok && w.next(a, deal));
        }
        return;
    }

    const int g = lane >> 2, t = lane & 3;
    const int key0 = warp * 16 + g, key1 = key0 + 8;                     // this lane's keys of a unit, for the scores
    // where in a stage this lane's words are
    const uint32_t base = smem_u32(stages);
    auto word = [](int row, int chunk) {                                 // byte of a 16-byte chunk in the swizzled block
        return D == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    };
    uint32_t k_at[2][WK], v_at[4];
#pragma unroll
    for (int j = 0; j < WK; ++j) { k_at[0][j] = word(key0, t * WK + j); k_at[1][j] = word(key1, t * WK + j); }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = warp * 16 + 2 * t + (j & 1) + (j >> 1) * 8;
        v_at[j] = BLOCK * D + (D == 128 ? word(row, g) : word(row, g >> 1) + (g & 1) * 8);
    }
    int q_token[NT], token[NT][2];                                       // of this lane's row of the queries, and of its two rows of the scores
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        q_token[nt] = (nt * 8 + g) / deal.group;
        token[nt][0] = (nt * 8 + 2 * t) / deal.group;
        token[nt][1] = (nt * 8 + 2 * t + 1) / deal.group;
    }
    uint32_t q[NT][KS][2];
    auto load_queries = [&](const Walk& w, uint32_t (&q)[NT][KS][2]) {   // rows that are not there are zeros
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const bool live = q_token[nt] < w.sp.n;
            const __half* src = a.q + (size_t)(w.sp.row + min(q_token[nt], w.sp.n - 1)) * a.ldq +
                                (w.head * deal.group + nt * 8 + g - q_token[nt] * deal.group) * D + t * (D / 4);
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const uint4 v = live ? reinterpret_cast<const uint4*>(src)[j] : make_uint4(0, 0, 0, 0);
                q[nt][2 * j][0] = v.x; q[nt][2 * j][1] = v.y;
                q[nt][2 * j + 1][0] = v.z; q[nt][2 * j + 1][1] = v.w;
            }
        }
    };
    load_queries(w, q);

    int i = 0;
    for (bool more = true; more;) {                                      // a warp whose wait ran out goes on to the end, so that all meet at the barriers
        const int first = w.sp.pos, last = w.sp.pos + w.sp.n - 1, length = last + 1, held = length / BLOCK;
        const size_t at = (size_t)w.seq * a.c.kv_heads + w.head;
        const float* k_scale = a.c.k_scale + at * (a.c.capacity / BLOCK);
        const float* v_scale = a.c.v_scale + at * (a.c.capacity / BLOCK);
        float ks = w.u0 < held ? k_scale[w.u0] : 1.0f, vs = w.u0 < held ? v_scale[w.u0] : 1.0f;
        float o[KS][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[mt][nt][c] = 0.0f;
        }
        for (int u = w.u0; u < w.u0 + w.n; ++u) {
            float s[2][NT][4];                                           // two sums, so that a product waits for the one before the last
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[0][nt][c] = s[1][nt][c] = 0.0f;
            uint32_t vw[4][DPL / 4];                                     // codes of this lane's elements of four keys
            const float factor = a.scale * LOG2E * ks;
            float inv = power_of_two(-exponent_of(vs)), ev = (float)exponent_of(vs);
            if (u + 1 < w.u0 + w.n) { ks = u + 1 < held ? k_scale[u + 1] : 1.0f; vs = u + 1 < held ? v_scale[u + 1] : 1.0f; }
            const bool codes = u < held;
            const int valid = length - u * BLOCK;                        // tokens of the tail that are there; what lies behind them is taken as zeros
            const uint32_t src = base + i % F::STAGES * F::STAGE;
            tc::wait_uniform(&full[i % F::STAGES], (uint32_t)(i / F::STAGES) & 1u, abort_flag);
            if (codes) {
                uint4 kw[2][WK];
#pragma unroll
                for (int j = 0; j < WK; ++j)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(kw[k][j].x), "=r"(kw[k][j].y), "=r"(kw[k][j].z), "=r"(kw[k][j].w)
                                     : "r"(src + k_at[k][j]));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (D == 128)
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(vw[j][0]), "=r"(vw[j][1]), "=r"(vw[j][2]), "=r"(vw[j][3]) : "r"(src + v_at[j]));
                    else
                        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(vw[j][0]), "=r"(vw[j][1]) : "r"(src + v_at[j]));
                }
#pragma unroll
                for (int j = 0; j < WK; ++j) {
                    const uint32_t x[4] = {kw[0][j].x, kw[0][j].y, kw[0][j].z, kw[0][j].w}, y[4] = {kw[1][j].x, kw[1][j].y, kw[1][j].z, kw[1][j].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t a0 = codes_f16(x[k]), a1 = codes_f16(y[k]), a2 = codes_f16_hi(x[k]), a3 = codes_f16_hi(y[k]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16x8x16(s[k & 1][nt], a0, a1, a2, a3, q[nt][j * 4 + k][0], q[nt][j * 4 + k][1]);
                    }
                }
                if (ev == 0.0f) {                                        // that of zeros too
                    uint32_t any = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int k = 0; k < DPL / 4; ++k) any |= vw[j][k];
                    if (!__any_sync(0xffffffffu, (any & 0x7f7f7f7fu) != 0)) { ev = (float)NO_VALUES; inv = power_of_two(-NO_VALUES); }
                }
            } else {
                const uint8_t* kt = stages + i % F::STAGES * F::STAGE;
                const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint4 x = key0 < valid ? reinterpret_cast<const uint4*>(kt + key0 * D * 2 + t * (D / 2))[j] : none;
                    const uint4 y = key1 < valid ? reinterpret_cast<const uint4*>(kt + key1 * D * 2 + t * (D / 2))[j] : none;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16x8x16(s[0][nt], x.x, y.x, x.y, y.y, q[nt][2 * j][0], q[nt][2 * j][1]);
                        mma_16x8x16(s[1][nt], x.z, y.z, x.w, y.w, q[nt][2 * j + 1][0], q[nt][2 * j + 1][1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[i % F::STAGES]);
                ++i;
                tc::wait_uniform(&full[i % F::STAGES], (uint32_t)(i / F::STAGES) & 1u, abort_flag);
            }
            // exponents, masked where not every row sees every key of the unit
            const bool all_seen = (u + 1) * BLOCK - 1 <= first && last - u * BLOCK < a.window;
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float x = fmaf(s[0][nt][c] + s[1][nt][c], factor, ev);
                    if (!all_seen) {
                        const int key = u * BLOCK + (c < 2 ? key0 : key1), p = first + min(token[nt][c & 1], w.sp.n - 1);
                        if (!(key <= p && p - key < a.window)) x = -INFINITY;
                    }
                    s[0][nt][c] = x;
                    over |= x > m[nt][c & 1] + MOST_TOP;
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        top -= LEAST_TOP;
                        if (top > m[nt][c]) {
                            const float before = ex2(m[nt][c] - top);
                            m[nt][c] = top;
                            l[nt][c] *= before;
#pragma unroll
                            for (int mt = 0; mt < KS; ++mt) { o[mt][nt][c] *= before; o[mt][nt][c + 2] *= before; }
                        }
                    }
            }
            uint32_t p[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) e[c] = ex2(s[0][nt][c] - (m[nt][c & 1] == -INFINITY ? 0.0f : m[nt][c & 1]));
                l[nt][0] = fmaf(e[0] + e[2], inv, l[nt][0]);
                l[nt][1] = fmaf(e[1] + e[3], inv, l[nt][1]);
                p[nt][0] = transposed_8x8(pack_f16(e[0], e[1]));
                p[nt][1] = transposed_8x8(pack_f16(e[2], e[3]));
            }
            if (codes) {
#pragma unroll
                for (int k = 0; k < DPL / 4; ++k) {                      // four elements: two m-tiles
                    const uint32_t lo0 = __byte_perm(vw[0][k], vw[1][k], 0x5140), hi0 = __byte_perm(vw[0][k], vw[1][k], 0x7362);
                    const uint32_t lo1 = __byte_perm(vw[2][k], vw[3][k], 0x5140), hi1 = __byte_perm(vw[2][k], vw[3][k], 0x7362);
                    const uint32_t a0 = codes_f16(lo0), a1 = codes_f16_hi(lo0), a2 = codes_f16(lo1), a3 = codes_f16_hi(lo1);
                    const uint32_t b0 = codes_f16(hi0), b1 = codes_f16_hi(hi0), b2 = codes_f16(hi1), b3 = codes_f16_hi(hi1);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16x8x16(o[2 * k][nt], a0, a1, a2, a3, p[nt][0], p[nt][1]);
                        mma_16x8x16(o[2 * k + 1][nt], b0, b1, b2, b3, p[nt][0], p[nt][1]);
                    }
                }
            } else {
                const uint8_t* vt = stages + i % F::STAGES * F::STAGE;
                const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < DPL / 8; ++k) {                      // eight elements: four m-tiles
                    uint4 x[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int row = warp * 16 + 2 * t + (j & 1) + (j >> 1) * 8;
                        x[j] = row < valid ? reinterpret_cast<const uint4*>(vt + row * D * 2 + g * DPL * 2)[k] : none;
                    }
                    const uint32_t y[4][4] = {{x[0].x, x[1].x, x[2].x, x[3].x}, {x[0].y, x[1].y, x[2].y, x[3].y}, {x[0].z, x[1].z, x[2].z, x[3].z}, {x[0].w, x[1].w, x[2].w, x[3].w}};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t a0 = __byte_perm(y[e][0], y[e][1], 0x5410), a1 = __byte_perm(y[e][0], y[e][1], 0x7632);
                        const uint32_t a2 = __byte_perm(y[e][2], y[e][3], 0x5410), a3 = __byte_perm(y[e][2], y[e][3], 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16x8x16(o[4 * k + e][nt], a0, a1, a2, a3, p[nt][0], p[nt][1]);
                    }
                }
            }
            // Not ahead of the products: words that were only asked for were overtaken by the next copy in a call of forty.
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[i % F::STAGES]);
            ++i;
        }
        // ---- the next tile's queries are asked for, then the four warps' parts of this one are added up ----
        const int rows = w.sp.n * deal.group;
        const bool alone = w.begins && w.ends;
        float* part = a.partial + (2 * (size_t)blockIdx.x + (w.begins ? 1 : 0)) * partial_floats(F::TILE, D);
        __half* out = a.out + (size_t)w.sp.row * a.ldo + w.head * deal.group * D;
        more = w.next(a, deal);
        if (more) load_queries(w, q);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
        named_bar_sync(1, 32 * FEW_WARPS);                               // the tile before has been read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = nt * 8 + 2 * t + c;
                if (g == 0) { s_m[warp][r] = m[nt][c]; s_l[warp][r] = l[nt][c]; }
                float4* row = join + (warp * F::TILE + r) * (D / 4);     // this lane's elements, DPL of them: m-tile mt has 2 mt and 2 mt + 1
#pragma unroll
                for (int j = 0; j < DPL / 4; ++j)
                    row[(g * (DPL / 4) + j) ^ t] = make_float4(o[2 * j][nt][c], o[2 * j][nt][c + 2], o[2 * j + 1][nt][c], o[2 * j + 1][nt][c + 2]);
            }
        named_bar_sync(1, 32 * FEW_WARPS);
        const bool ok = *abort_flag == 0;
        for (int j = tid; j < rows * (D / 4); j += 32 * FEW_WARPS) {
            const int r = j / (D / 4), d = j % (D / 4);
            const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r])), ref = top == -INFINITY ? 0.0f : top;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.0f;
#pragma unroll
            for (int x = 0; x < FEW_WARPS; ++x) {                        // in warp order; a NaN sum stays one
                const float f = ex2(s_m[x][r] - ref);
                const float4 y = join[(x * F::TILE + r) * (D / 4) + (d ^ ((r >> 1) & 3))];
                v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
                sum = fmaf(s_l[x][r], f, sum);
            }
            if (!ok) continue;
            if (alone) {
                const float n = 1.0f / sum;
                const int i_token = r / deal.group;
                *reinterpret_cast<uint2*>(out + (size_t)i_token * a.ldo + (r - i_token * deal.group) * D + d * 4) =
                    make_uint2(pack_f16(v.x * n, v.y * n), pack_f16(v.z * n, v.w * n));
            } else {
                reinterpret_cast<float4*>(part + r * D)[d] = v;
                if (d == 0) { part[F::TILE * D + r] = top; part[F::TILE * (D + 1) + r] = sum; }
            }
        }
    }
    if (tid == 0) leave_word(a, deal, w, start);
}

// ------------------------------------------------------------------------------------------------------------- merge --
// Joins the tiles that several CTAs have keys of: CTA x takes the tile that CTA x of the kernel before began and did not end.  Its parts are
// the last part of that CTA and the first parts of those behind it; the same call adds them up in the same order.
// A row is LANES threads, four elements each; SIDES groups of them share a row's parts: where there are few rows, there are many parts.  Bound by
// latency, that of the launch of CTAs without a tile among it (us of a call with 256 threads and eight groups, 128 and four, 128 and two: 500
// tokens 8.7, 7.8, 7.5; 2049 tokens 9.1, 8.6, 9.0; 100 000 tokens 25.7, 26.4, 29.5; 96 sequences 121.4, 119.0, 117.9).
constexpr int MERGE_THREADS = 128, SIDES = 4;
template <int D>
__global__ void __launch_bounds__(MERGE_THREADS)
merge_kernel(const __grid_constant__ AttnArgs a, int tile)
{
    constexpr int LANES = D / 4, ROWS = MERGE_THREADS / (LANES * SIDES);         // rows of a CTA
    __shared__ float4 red[SIDES][ROWS][LANES];
    __shared__ float2 red_ml[SIDES][ROWS];
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const Join w = a.joins[blockIdx.x];
    if ((int)blockIdx.y * ROWS >= w.rows || w.parts == 0) return;
    const int lane = threadIdx.x % LANES, mine = threadIdx.x / LANES % ROWS, side = threadIdx.x / (LANES * ROWS);
    const int r = min((int)blockIdx.y * ROWS + mine, w.rows - 1);
    const size_t each = partial_floats(tile, D);
    const float* base = a.partial + (2 * (size_t)blockIdx.x + 1) * each;         // part j > 0: the first of CTA x + j
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, l = 0.0f;
    constexpr int AT_ONCE = 4;
    for (int j0 = side; j0 < w.parts; j0 += AT_ONCE * SIDES) {
        float4 x[AT_ONCE];
        float m[AT_ONCE], n[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int j = j0 + i * SIDES;
            const float* p = j == 0 ? base : base + (2 * (size_t)j - 1) * each;
            const bool there = j < w.parts;
            x[i] = there ? reinterpret_cast<const float4*>(p + r * D)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
            m[i] = there ? p[tile * D + r] : -INFINITY;
            n[i] = there ? p[tile * (D + 1) + r] : 0.0f;
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) now = fmaxf(now, m[i]);
        const float ref = now == -INFINITY ? 0.0f : now;
        const float f = ex2(top - ref);
        v.x *= f; v.y *= f; v.z *= f; v.w *= f;
        l *= f;
        top = now;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const float g = ex2(m[i] - ref);
            v.x = fmaf(x[i].x, g, v.x); v.y = fmaf(x[i].y, g, v.y); v.z = fmaf(x[i].z, g, v.z); v.w = fmaf(x[i].w, g, v.w);
            l = fmaf(n[i], g, l);
        }
    }
    red[side][mine][lane] = v;
    if (lane == 0) red_ml[side][mine] = make_float2(top, l);
    __syncthreads();
    if (side > 0) return;
    for (int x = 0; x < SIDES; ++x) top = fmaxf(top, red_ml[x][mine].x);
    const float ref = top == -INFINITY ? 0.0f : top;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.0f;
#pragma unroll
    for (int x = 0; x < SIDES; ++x) {
        const float2 ml = red_ml[x][mine];
        const float4 y = red[x][mine][lane];
        const float g = ex2(ml.x - ref);
        v.x = fmaf(y.x, g, v.x); v.y = fmaf(y.y, g, v.y); v.z = fmaf(y.z, g, v.z); v.w = fmaf(y.w, g, v.w);
        l = fmaf(ml.y, g, l);
    }
    if ((int)blockIdx.y * ROWS + mine >= w.rows) return;
    const float n = 1.0f / l;
    const int group = a.num_heads / a.c.kv_heads, row = w.row0 + r;
    __half* dst = a.out + (size_t)(w.row + row / group) * a.ldo + (w.head * group + row % group) * D + lane * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f16(v.x * n, v.y * n), pack_f16(v.z * n, v.w * n));
}

// The same for tiles of PROMPT_ROWS rows, which lie in the workspace by columns, [D / 4][rows] of four, as the kernel before has them: neighbouring
// threads take neighbouring rows, and 16 columns each; four parts' loads at once (a sequence of 60000 tokens, 64 rows of 28 heads on 4: one part after
// another 66.4 us of the whole, four at once 54.8).
constexpr int PROMPT_ROWS = 256, MERGE_ROWS = 32;
template <int D>
__global__ void __launch_bounds__(MERGE_ROWS * D / 16)
merge_columns_kernel(const __grid_constant__ AttnArgs a)
{
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const Join w = a.joins[blockIdx.x];
    const int r = blockIdx.y * MERGE_ROWS + threadIdx.x % MERGE_ROWS, c0 = threadIdx.x / MERGE_ROWS * 4;         // columns 4 c0 ... 4 c0 + 15
    if (w.parts == 0 || r >= w.rows) return;
    const size_t each = partial_floats(PROMPT_ROWS, D);
    const float* base = a.partial + (2 * (size_t)blockIdx.x + 1) * each;         // part j > 0: the first of CTA x + j
    float4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, l = 0.0f;
    constexpr int AT_ONCE = 4;
    for (int j0 = 0; j0 < w.parts; j0 += AT_ONCE) {
        float4 x[AT_ONCE][4];
        float m[AT_ONCE], n[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int j = j0 + i;
            const float* p = j == 0 ? base : base + (2 * (size_t)j - 1) * each;
            const bool there = j < w.parts;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[i][c] = there ? reinterpret_cast<const float4*>(p)[(c0 + c) * PROMPT_ROWS + r] : make_float4(0.f, 0.f, 0.f, 0.f);
            m[i] = there ? p[PROMPT_ROWS * D + r] : -INFINITY;
            n[i] = there ? p[PROMPT_ROWS * (D + 1) + r] : 0.0f;
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) now = fmaxf(now, m[i]);
        const float ref = now == -INFINITY ? 0.0f : now, f = ex2(top - ref);
        top = now;
        l *= f;
#pragma unroll
        for (int c = 0; c < 4; ++c) { v[c].x *= f; v[c].y *= f; v[c].z *= f; v[c].w *= f; }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const float g = ex2(m[i] - ref);
            l = fmaf(n[i], g, l);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c].x = fmaf(x[i][c].x, g, v[c].x); v[c].y = fmaf(x[i][c].y, g, v[c].y);
                v[c].z = fmaf(x[i][c].z, g, v[c].z); v[c].w = fmaf(x[i][c].w, g, v[c].w);
            }
        }
    }
    const float n = 1.0f / l;
    const int group = a.num_heads / a.c.kv_heads, row = w.row0 + r;
    uint4* dst = reinterpret_cast<uint4*>(a.out + (size_t)(w.row + row / group) * a.ldo + (w.head * group + row % group) * D + c0 * 4);
#pragma unroll
    for (int c = 0; c < 4; c += 2)
        dst[c / 2] = make_uint4(pack_f16(v[c].x * n, v[c].y * n), pack_f16(v[c].z * n, v[c].w * n), pack_f16(v[c + 1].x * n, v[c + 1].y * n),
                                pack_f16(v[c + 1].z * n, v[c + 1].w * n));
}

}  // namespace cache8
}  // namespace twm
