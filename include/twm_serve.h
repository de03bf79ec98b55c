/*
 * twm_serve.h — what a serving decode step needs beside twm_decode.h: a key/value cache held in 8 bits with the
 * append that fills it and the attention that reads it, and sampling.  Same conventions as twmarlin.h: device pointers
 * owned by the caller, enqueue only, nothing allocated, status returned.  `flags` takes TWM_FLAG_PDL as twm_decode.h does:
 * the kernels wait for the one before ahead of reading anything that they use.
 *
 * The cache.  Sequence s, key/value head h: blocks of 64 tokens.  A full block is held as e4m3 codes and one power of two
 * each for its keys and its values: value = code * 2^e, e the smallest integer with amax <= 448 * 2^e, amax over the
 * block's finite FP16 values (a block of zeros has scale 1).  The FP16 values are rounded once, when the block is
 * full.  The tokens of a block that is not full stay FP16: `tail` holds two blocks, block b in half b & 1.  An infinite or NaN
 * element of a key is held as NaN; one of a value as zero, and the first element of its key as NaN: every row that
 * sees the token is NaN in that head, and no other row is.  So what the cache holds does not depend on the portions in which tokens came,
 * and a sequence can be cut back to any length >= 64 * (ceil(longest / 64) - 2), longest the most tokens it has held, by
 * appending there next.
 *
 * The rows of a call.  Sequence s of the cache has the rows row_start[s] <= r < row_start[s + 1] of the call (device
 * array of seqs + 1; NULL: one row each, rows == seqs and max_rows == 1), `max_rows` of them at most (1 <= max_rows <= rows); its first row is at position start[s]
 * (device array of seqs), which is the number of tokens cached before the step.  start[s] < 0 takes the sequence out of the call.
 * Rows behind row_start[seqs], and rows at positions past the capacity, are left as they were.
 */
#ifndef TWM_SERVE_H
#define TWM_SERVE_H

#include "twmarlin.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { TWM_BF16 = 2 };           /* beside TWM_F32 and TWM_F16 */
enum { TWM_CACHE8_BLOCK = 64 };  /* tokens of a block */

typedef struct twm_cache8 {
    int seqs, kv_heads;
    int head_dim;                /* 64 or 128 */
    int capacity;                /* tokens per sequence, a multiple of 64 */
    void* k;                     /* e4m3 [seqs][kv_heads][capacity][head_dim] */
    void* v;
    float* k_scale;              /* [seqs][kv_heads][capacity / 64] */
    float* v_scale;
    void* k_tail;                /* f16 [seqs][kv_heads][2][64][head_dim] */
    void* v_tail;
} twm_cache8;

/* Bias and rotate-half RoPE on q and k, bias on v, k and v appended; qkv is the fused QKV output [rows][q | k | v] (f16, row
 * stride ldqkv), q_out the rotated queries [rows][q] (f16, row stride ldq).  rope_table: f32 [capacity][head_dim], cosines then
 * sines of every position, or NULL for none; bias: f32 [q | k | v] or NULL.  What twm_rope_append is to the FP16 cache.
 * q_out may be the q columns of qkv themselves, and overlaps qkv in no other way (refused).  Pointers on 16 bytes, row strides multiples of 8. */
typedef struct twm_cache8_append_args {
    void* q_out;
    long ldq;
    const void* qkv;
    long ldqkv;
    const float* bias;
    const float* rope_table;
    int num_heads;
    int rows, max_rows;
    const int* row_start;
    const int* start;
} twm_cache8_append_args;
twm_status twm_cache8_append(const twm_cache8* cache, const twm_cache8_append_args* args, int flags, void* stream);

/* Bytes of workspace twm_cache8_attention needs.  Nothing in it is kept from call to call. */
size_t twm_cache8_attention_bytes(const twm_cache8* cache, int num_heads, int max_rows);

/* Softmax attention of the rows of a call over the cache, which already holds their own keys and values: the row at position p
 * sees the keys j <= p with p - j < window (window 0: all).  A sequence taken out of the call gets zeros.
 * out and q: f16 [rows][num_heads * head_dim], row strides ldo and ldq; query head h reads key/value head
 * h / (num_heads / kv_heads); scale is positive.  out must not overlap q (refused).  Pointers on 16 bytes, row strides multiples of 8.
 * Calls that share a workspace must not overlap. */
typedef struct twm_cache8_attention_args {
    void* out;
    long ldo;
    const void* q;
    long ldq;
    int num_heads;
    int rows, max_rows;
    int window;
    const int* row_start;
    const int* start;
    void* workspace;
    size_t workspace_bytes;
    float scale;
} twm_cache8_attention_args;
twm_status twm_cache8_attention(const twm_cache8* cache, const twm_cache8_attention_args* args, int flags, void* stream);

/* One token of every row of logits.  With w_i = exp((l_i - max l) / temperature) and the order of falling l, equal ones by
 * rising index:
 *   top_k   the first top_k of the order are kept (<= 0: all);
 *   top_p   of these the shortest head of the order that holds top_p of their sum of w (>= 1: all; the first one always);
 *   min_p   of these the ones with w >= min_p (<= 0: all; values over 1 count as 1).
 * The token is the first index, rising, at which the running sum of the kept w exceeds random * their sum; prob is its w over
 * that sum.  temperature 0 (or not > 0): the first largest logit; +inf: all finite logits weigh the same.  A NaN logit counts as -inf; a row without any other gives
 * token 0.  Sums do not depend on an order: the same call gives the same token. */
typedef struct twm_sample_args {
    int rows, vocab;             /* vocab: at most 2^20 */
    int dtype;                   /* TWM_F32, TWM_F16 or TWM_BF16 */
    const void* logits;          /* [rows], row stride ld */
    long ld;
    const float* random;         /* [rows], each in [0, 1); with `step`: [random_count], see there */
    const float* temperature;    /* [rows]; NULL = 1 */
    const int* top_k;            /* [rows]; NULL = all */
    const float* top_p;          /* [rows]; NULL = all */
    const float* min_p;          /* [rows]; NULL = all */
    int* tokens;                 /* [rows] */
    float* prob;                 /* [rows] or NULL */
    /* Decode loop of one row, as twm_argmax_advance: with step != NULL (then rows == 1 and pos and len are there too) the random
     * number is random[min(step[0], random_count - 1)], history[step[0]] = token when it fits (history may be NULL), and step[0],
     * pos[0] and len[0] advance by one. */
    int* step;
    int random_count;
    int* history;
    int history_capacity;
    int* pos;
    int* len;
} twm_sample_args;

twm_status twm_sample(const twm_sample_args* args, int flags, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TWM_SERVE_H */
