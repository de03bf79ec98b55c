// twm_serve.cuh — argument checks and launches of include/twm_serve.h.  Part of twmarlin.cu's translation unit.
#pragma once

#include <climits>

#include "twm_cache8.cuh"
#include "twm_cache8_attn.cuh"
#include "twm_sample.cuh"

namespace {

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// What both calls on a cache check: the cache itself and the rows.
twm_status check_cache8(const twm_cache8* c, int num_heads, int rows, const int* row_start, int max_rows, const int* start)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !start) return TWM_EINVAL;
    if (c->seqs < 1 || c->seqs > 65535 || c->kv_heads < 1 || c->kv_heads > 65535 || (c->head_dim != 64 && c->head_dim != 128)) return TWM_EINVAL;
    if (c->capacity < TWM_CACHE8_BLOCK || c->capacity % TWM_CACHE8_BLOCK) return TWM_EINVAL;
    // tensor maps and row numbers count cached rows in 32 bits
    if ((long long)c->seqs * c->kv_heads * c->capacity > INT_MAX) return TWM_EINVAL;
    if (num_heads < 1 || num_heads % c->kv_heads || rows < 1 || max_rows < 1 || max_rows > rows) return TWM_EINVAL;
    if (!row_start && (rows != c->seqs || max_rows != 1)) return TWM_EINVAL;
    if ((long long)num_heads * c->head_dim > (1 << 20) || (long long)max_rows * num_heads > INT_MAX / 2) return TWM_EINVAL;
    if (off16(c->k) || off16(c->v) || off16(c->k_tail) || off16(c->v_tail)) return TWM_EALIGN;
    return TWM_OK;
}
twm::cache8::Cache device_cache(const twm_cache8* c)
{
    return {c->seqs, c->kv_heads, c->capacity, (uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, (__half*)c->k_tail, (__half*)c->v_tail};
}

}  // namespace

extern "C" {

twm_status twm_cache8_append(const twm_cache8* cache, void* q_out, long ldq, const void* qkv, long ldqkv, const float* bias,
                             const float* rope_table, int num_heads, int rows, const int* row_start, int max_rows, const int* start,
                             int flags, void* stream)
{
    twm_status st = check_cache8(cache, num_heads, rows, row_start, max_rows, start);
    if (st == TWM_EINVAL) return st;
    if (!q_out || !qkv || ldq < (long)num_heads * cache->head_dim || ldqkv < (long)(num_heads + 2 * cache->kv_heads) * cache->head_dim) return TWM_EINVAL;
    if (st != TWM_OK) return st;
    if (off16(q_out) || off16(qkv) || off16(bias) || off16(rope_table) || (ldq & 7) || (ldqkv & 7)) return TWM_EALIGN;
    if ((st = ensure_device(nullptr)) != TWM_OK) return st;
    const twm::cache8::AppendArgs a = {device_cache(cache), {row_start, start, rows, max_rows}, (__half*)q_out, (const __half*)qkv, bias, rope_table,
                                       ldq, ldqkv, num_heads};
    // blocks that max_rows tokens can touch, wherever they begin
    const dim3 grid((unsigned)(((long)max_rows + 2 * TWM_CACHE8_BLOCK - 2) / TWM_CACHE8_BLOCK), cache->kv_heads, cache->seqs);
    return launch_op("twm_cache8_append", cache->head_dim == 64 ? twm::cache8::append_kernel<64> : twm::cache8::append_kernel<128>, grid,
                     dim3(twm::cache8::APPEND_THREADS), 0, flags, stream, a);
}

size_t twm_cache8_attention_bytes(const twm_cache8* c, int num_heads, int max_rows)
{
    if (!c || num_heads < 1 || max_rows < 1 || c->seqs < 1 || c->kv_heads < 1 || (c->head_dim != 64 && c->head_dim != 128)) return 0;
    return 16;
}

twm_status twm_cache8_attention(const twm_cache8* cache, void* out, long ldo, const void* q, long ldq, int num_heads, int rows, const int* row_start,
                                int max_rows, const int* start, float scale, int window, void* workspace, size_t workspace_bytes, int flags,
                                void* stream)
{
    twm_status st = check_cache8(cache, num_heads, rows, row_start, max_rows, start);
    if (st == TWM_EINVAL) return st;
    if (!out || !q || !workspace || window < 0 || !(scale > 0.0f) || ldo < (long)num_heads * cache->head_dim || ldq < (long)num_heads * cache->head_dim)
        return TWM_EINVAL;
    if (st != TWM_OK) return st;
    if (off16(out) || off16(q) || off16(workspace) || (ldo & 7) || (ldq & 7)) return TWM_EALIGN;
    if (workspace_bytes < twm_cache8_attention_bytes(cache, num_heads, max_rows)) return TWM_EWORKSPACE;
    if ((st = ensure_device(nullptr)) != TWM_OK) return st;
    const twm::cache8::AttnArgs a = {device_cache(cache), {row_start, start, rows, max_rows}, (__half*)out, (const __half*)q, ldo, ldq, num_heads,
                                     window ? window : INT_MAX, scale};
    const dim3 grid((unsigned)(((long)max_rows * num_heads + 3) / 4), cache->seqs);
    return launch_op("twm_cache8_attention", cache->head_dim == 64 ? twm::cache8::attn_plain_kernel<64> : twm::cache8::attn_plain_kernel<128>, grid,
                     dim3(twm::cache8::PLAIN_THREADS), 0, flags, stream, a);
}

twm_status twm_sample(const twm_sample_args* args, int flags, void* stream)
{
    if (!args || !args->logits || !args->random || !args->tokens || args->rows < 1 || args->vocab < 1 || args->ld < args->vocab) return TWM_EINVAL;
    if (args->dtype != TWM_F32 && args->dtype != TWM_F16 && args->dtype != TWM_BF16) return TWM_EINVAL;
    if (args->step && (args->rows != 1 || args->random_count < 1 || !args->pos || !args->len || (args->history && args->history_capacity < 1)))
        return TWM_EINVAL;
    if (reinterpret_cast<uintptr_t>(args->logits) & (args->dtype == TWM_F32 ? 3 : 1)) return TWM_EALIGN;
    const twm_status st = ensure_device(nullptr);
    if (st != TWM_OK) return st;
    auto* kernel = args->dtype == TWM_F32   ? twm::sample::sample_kernel<float>
                   : args->dtype == TWM_F16 ? twm::sample::sample_kernel<__half>
                                            : twm::sample::sample_kernel<__nv_bfloat16>;
    return launch_op("twm_sample", kernel, dim3(args->rows), dim3(twm::sample::THREADS), 0, flags, stream, *args);
}

}  // extern "C"
