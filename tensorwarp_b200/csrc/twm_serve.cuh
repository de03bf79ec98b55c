// twm_serve.cuh — argument checks and launches of include/twm_serve.h.  Part of twmarlin.cu's translation unit.
#pragma once

#include <atomic>
#include <climits>
#include <cmath>

#include "twm_cache8.cuh"
#include "twm_cache8_attn.cuh"
#include "twm_cache8_prompt.cuh"
#include "twm_sample.cuh"

namespace {

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// What both calls on a cache check: the cache itself and the rows.
twm_status check_cache8(const twm_cache8* c, int num_heads, int rows, const int* row_start, int max_rows, const int* start)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !start) return TWM_EINVAL;
    if (c->seqs < 1 || c->seqs > 65535 || c->kv_heads < 1 || c->kv_heads > 4096 || (c->head_dim != 64 && c->head_dim != 128)) return TWM_EINVAL;
    if (c->capacity < TWM_CACHE8_BLOCK || c->capacity % TWM_CACHE8_BLOCK) return TWM_EINVAL;
    // tensor maps and row numbers count cached rows in 32 bits
    if ((long long)c->seqs * c->kv_heads * c->capacity > INT_MAX) return TWM_EINVAL;
    if (num_heads < 1 || num_heads > 4096 || num_heads % c->kv_heads || rows < 1 || max_rows < 1 || max_rows > rows) return TWM_EINVAL;
    if (!row_start && (rows != c->seqs || max_rows != 1)) return TWM_EINVAL;
    if ((long long)num_heads * c->head_dim > (1 << 20) || (long long)max_rows * num_heads > INT_MAX / 2) return TWM_EINVAL;
    if (off16(c->k) || off16(c->v) || off16(c->k_tail) || off16(c->v_tail)) return TWM_EALIGN;
    return TWM_OK;
}
// Whether two lots of FP16 rows, of `wa` and `wb` numbers, have memory in common.  Columns of one buffer have none, though they lie in one another's range.
bool rows_overlap(const void* a, long lda, long wa, const void* b, long ldb, long wb, int rows)
{
    typedef long long ll;
    const ll x0 = (ll)reinterpret_cast<uintptr_t>(a), y0 = (ll)reinterpret_cast<uintptr_t>(b), sx = 2 * (ll)lda, sy = 2 * (ll)ldb, nx = 2 * (ll)wa, ny = 2 * (ll)wb;
    if (x0 + (rows - 1) * sx + nx <= y0 || y0 + (rows - 1) * sy + ny <= x0) return false;
    // of equal strides the first and the last row show what all others do
    for (ll i = 0; i < rows; i += lda == ldb ? std::max(rows - 1, 1) : 1) {
        const ll x = x0 + i * sx, behind = x - ny - y0;                  // the first of b's rows that ends behind x
        const ll j = behind < 0 ? 0 : behind / sy + 1;
        if (j < rows && y0 + j * sy < x + nx) return true;
    }
    return false;
}
twm::cache8::Cache device_cache(const twm_cache8* c)
{
    return {c->seqs, c->kv_heads, c->capacity, (uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, (__half*)c->k_tail, (__half*)c->v_tail};
}

// How attention is launched: the rows of a tile, how many of them there can be, and the CTAs of the grid, whatever the lengths (which are on the device).
// Up to 16 rows the kernel for few is the faster one, though it spills with more than 8 of heads of 128 (us, and those of the kernel for many: 96
// sequences of 4000 tokens, 40 heads on 8, 10 rows 257 and 357, 15 rows 264 and 357; 16 heads on 1, 16 rows 52 and 60; one sequence of 2048, 14 rows
// 13.7 and 16.6; 40 of 3000, heads of 64, 16 rows 50 and 104).  It has no form for more; the other takes 361 us for 20 rows of the first batch, and
// 71 us (1.9 TB/s) for 64 sequences of 8000 tokens with 71 heads on 1.
struct AttnPlan { int tile, rows, ctas; };
AttnPlan plan_attention(int group, int max_rows, int head_dim)
{
    const long rows = (long)max_rows * group;
    if (rows <= 8) return {8, (int)rows, kDefaultSms * (head_dim == 64 ? twm::cache8::Few<64, 1>::CTAS : twm::cache8::Few<128, 1>::CTAS)};
    if (rows <= 16) return {16, (int)rows, kDefaultSms * (head_dim == 64 ? twm::cache8::Few<64, 2>::CTAS : twm::cache8::Few<128, 2>::CTAS)};
    return {twm::cache8::PROMPT_ROWS, (int)std::min(rows, (long)twm::cache8::PROMPT_ROWS), kDefaultSms};
}

// The codes of keys or values as [cached rows][head_dim], a box a block, swizzled over its whole row.
bool make_codes_map(CUtensorMap* map, const twm_cache8* c, void* codes)
{
    EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return false;
    const cuuint64_t gdim[2] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->seqs * c->kv_heads * c->capacity};
    const cuuint64_t gstride[1] = {(cuuint64_t)c->head_dim};
    const cuuint32_t box[2] = {(cuuint32_t)c->head_dim, TWM_CACHE8_BLOCK};
    const cuuint32_t estride[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
               c->head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Lets a kernel take more than 48 KB of shared memory on the current device.  The limit belongs to the function: it is set once a device (`done`, a
// bit each), to what every launch of it asks for.
twm_status allow_shared(const char* name, const void* kernel, size_t bytes, std::atomic<unsigned long long>& done)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < 64 && (done.load() >> dev & 1)) return TWM_OK;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) {
        if (dev < 64) done |= 1ULL << dev;
        return TWM_OK;
    }
    set_error(name, e);
    return TWM_ELAUNCH;
}

template <int D, int NT>
twm_status launch_few(const twm::cache8::AttnArgs& a, const AttnPlan& p, int flags, void* stream)
{
    auto* kernel = twm::cache8::few_kernel<D, NT>;
    constexpr size_t smem = twm::cache8::Few<D, NT>::SMEM;
    static std::atomic<unsigned long long> done{0};
    const twm_status st = allow_shared("twm_cache8_attention", (const void*)kernel, smem, done);
    if (st != TWM_OK) return st;
    return launch_op("twm_cache8_attention", kernel, dim3(p.ctas), dim3(twm::cache8::FEW_THREADS), smem, flags, stream, a);
}

template <int D>
twm_status launch_prompt(const twm::cache8::AttnArgs& a, const AttnPlan& p, int flags, void* stream)
{
    auto* kernel = twm::cache8::prompt_kernel<D>;
    constexpr size_t smem = twm::cache8::Prompt<D>::SMEM;
    static_assert(smem + 1024 < 227 * 1024, "shared memory of a CTA");
    static std::atomic<unsigned long long> done{0};
    const twm_status st = allow_shared("twm_cache8_attention", (const void*)kernel, smem, done);
    if (st != TWM_OK) return st;
    return launch_op("twm_cache8_attention", kernel, dim3(p.ctas), dim3(twm::cache8::PROMPT_THREADS), smem, flags, stream, a);
}

// Behind the kernel before whatever the flags: it waits for all of that one.
template <int D>
twm_status launch_merge(const twm::cache8::AttnArgs& a, const AttnPlan& p, int flags, void* stream)
{
    flags |= TWM_FLAG_PDL;
    if (p.tile == twm::cache8::PROMPT_ROWS)
        return launch_op("twm_cache8_attention(merge)", twm::cache8::merge_columns_kernel<D>, dim3(p.ctas, (p.rows + twm::cache8::MERGE_ROWS - 1) / twm::cache8::MERGE_ROWS),
                         dim3(twm::cache8::MERGE_ROWS * D / 16), 0, flags, stream, a);
    const int each = twm::cache8::MERGE_THREADS / (D / 4) / twm::cache8::SIDES;
    return launch_op("twm_cache8_attention(merge)", twm::cache8::merge_kernel<D>, dim3(p.ctas, (p.rows + each - 1) / each),
                     dim3(twm::cache8::MERGE_THREADS), 0, flags, stream, a, p.tile);
}

}  // namespace

extern "C" {

twm_status twm_cache8_append(const twm_cache8* cache, const twm_cache8_append_args* x, int flags, void* stream)
{
    if (!x) return TWM_EINVAL;
    twm_status st = check_cache8(cache, x->num_heads, x->rows, x->row_start, x->max_rows, x->start);
    if (st == TWM_EINVAL) return st;
    if (!x->q_out || !x->qkv || x->ldq < (long)x->num_heads * cache->head_dim || x->ldqkv < (long)(x->num_heads + 2 * cache->kv_heads) * cache->head_dim)
        return TWM_EINVAL;
    if (st != TWM_OK) return st;
    if (off16(x->q_out) || off16(x->qkv) || off16(x->bias) || off16(x->rope_table) || (x->ldq & 7) || (x->ldqkv & 7)) return TWM_EALIGN;
    if (!(x->q_out == x->qkv && (x->ldq == x->ldqkv || x->rows == 1)) &&
        rows_overlap(x->q_out, x->ldq, (long)x->num_heads * cache->head_dim, x->qkv, x->ldqkv, (long)(x->num_heads + 2 * cache->kv_heads) * cache->head_dim, x->rows))
        return TWM_EINVAL;
    if ((st = ensure_device(nullptr)) != TWM_OK) return st;
    const twm::cache8::AppendArgs a = {device_cache(cache), {x->row_start, x->start, x->rows, x->max_rows}, (__half*)x->q_out, (const __half*)x->qkv, x->bias,
                                       x->rope_table, x->ldq, x->ldqkv, x->num_heads, x->max_rows >= TWM_CACHE8_BLOCK / 4 ? 1 : 0};
    // blocks that max_rows tokens can touch, wherever they begin
    const dim3 grid((unsigned)(((long)x->max_rows + 2 * TWM_CACHE8_BLOCK - 2) / TWM_CACHE8_BLOCK), cache->kv_heads + (a.apart ? x->num_heads : 0), cache->seqs);
    return launch_op("twm_cache8_append", cache->head_dim == 64 ? twm::cache8::append_kernel<64> : twm::cache8::append_kernel<128>, grid,
                     dim3(twm::cache8::APPEND_THREADS), 0, flags, stream, a);
}

size_t twm_cache8_attention_bytes(const twm_cache8* c, int num_heads, int max_rows)
{
    if (!c || num_heads < 1 || max_rows < 1 || c->kv_heads < 1 || num_heads % c->kv_heads || (c->head_dim != 64 && c->head_dim != 128)) return 0;
    const AttnPlan p = plan_attention(num_heads / c->kv_heads, max_rows, c->head_dim);
    return (size_t)p.ctas * (sizeof(twm::cache8::Join) + 2 * twm::cache8::partial_floats(p.tile, c->head_dim) * sizeof(float));
}

twm_status twm_cache8_attention(const twm_cache8* cache, const twm_cache8_attention_args* x, int flags, void* stream)
{
    if (!x) return TWM_EINVAL;
    twm_status st = check_cache8(cache, x->num_heads, x->rows, x->row_start, x->max_rows, x->start);
    if (st == TWM_EINVAL) return st;
    const int D = cache->head_dim;
    if (!x->out || !x->q || !x->workspace || x->window < 0 || !(x->scale > 0.0f) || !(x->scale < INFINITY) || x->ldo < (long)x->num_heads * D ||
        x->ldq < (long)x->num_heads * D)
        return TWM_EINVAL;
    if (st != TWM_OK) return st;
    if (off16(x->out) || off16(x->q) || off16(x->workspace) || (x->ldo & 7) || (x->ldq & 7)) return TWM_EALIGN;
    if (rows_overlap(x->out, x->ldo, (long)x->num_heads * D, x->q, x->ldq, (long)x->num_heads * D, x->rows)) return TWM_EINVAL;
    if (x->workspace_bytes < twm_cache8_attention_bytes(cache, x->num_heads, x->max_rows)) return TWM_EWORKSPACE;
    if ((st = ensure_device(nullptr)) != TWM_OK) return st;
    const AttnPlan p = plan_attention(x->num_heads / cache->kv_heads, x->max_rows, D);
    auto* joins = (twm::cache8::Join*)x->workspace;
    twm::cache8::AttnArgs a = {device_cache(cache), {x->row_start, x->start, x->rows, x->max_rows}, (__half*)x->out, (const __half*)x->q, x->ldo, x->ldq,
                               x->num_heads, x->window ? x->window : INT_MAX, x->scale, joins, (float*)(joins + p.ctas), {}, {}};
    if (!make_codes_map(&a.k_map, cache, cache->k) || !make_codes_map(&a.v_map, cache, cache->v)) {
        snprintf(t_last_error, sizeof(t_last_error), "cuTensorMapEncodeTiled failed for a cache held in 8 bits");
        return TWM_ELAUNCH;
    }
    if (D == 64)
        st = p.tile == 8 ? launch_few<64, 1>(a, p, flags, stream) : p.tile == 16 ? launch_few<64, 2>(a, p, flags, stream) : launch_prompt<64>(a, p, flags, stream);
    else
        st = p.tile == 8 ? launch_few<128, 1>(a, p, flags, stream) : p.tile == 16 ? launch_few<128, 2>(a, p, flags, stream) : launch_prompt<128>(a, p, flags, stream);
    if (st != TWM_OK) return st;
    return D == 64 ? launch_merge<64>(a, p, flags, stream) : launch_merge<128>(a, p, flags, stream);
}

twm_status twm_sample(const twm_sample_args* args, int flags, void* stream)
{
    twm_status st = twm::sample::check(args);
    if (st != TWM_OK || (st = ensure_device(nullptr)) != TWM_OK) return st;
    const cudaError_t e = twm::sample::launch(*args, kDefaultSms, flags, stream);
    if (e == cudaSuccess) return TWM_OK;
    set_error("twm_sample", e);
    return TWM_ELAUNCH;
}

}  // extern "C"
