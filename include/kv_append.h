/*
 * Filling the paged caches on B200, C ABI: the step before every decode.
 *
 * For each new token: RMS norm of every q and k head (optional), rotation of
 * the first rotary_dim dims of every q and k head by the token's row of a
 * cosine / sine table (optional), and the write of its K and V to the page
 * the block table names, in one kernel.  The caches are the ones the decode
 * entry points read: gqa_decode.h (bf16 K and V pages), mla_decode.h (latent
 * pages) and kv4_decode.h (4-bit tiles).
 *
 * Tokens are rows of q, k and v.  Request b's new tokens are the rows
 * cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (cu_seqlens NULL: row b alone), and
 * seq_lens[b] counts its tokens AFTER the append, the value the decode that
 * follows takes: the last of its rows goes to position seq_lens[b] - 1.
 * Rows behind the last request and rows whose position is negative (a padded
 * batch: seq_lens[b] == 0) hold no token: nothing is written to the caches
 * for them, and their rows of q_out are zeroed when zero_skipped is set and
 * left as they were otherwise.  No two rows of one call may go to the same
 * page slot.
 *
 * The reference has no counterpart (its benchmarks fill the caches with
 * random data, bench/common.py:16-46).  Every launcher is asynchronous on
 * `stream`, allocates nothing, does not synchronise and can be captured into
 * a CUDA graph.  Pointers are device pointers; rows of 16-bit values and the
 * table are read in 16-byte pieces, so every base must be 16-byte aligned
 * and every stride a multiple of 8 elements.
 */
#ifndef KV_APPEND_B200_H
#define KV_APPEND_B200_H

#include <stddef.h>
#include <cuda_runtime_api.h>

#include "gqa_decode.h" /* gqa_bf16 */

#ifdef __cplusplus
extern "C" {
#endif

/* The new tokens and where they go. */
typedef struct kv_append_tokens {
  const int* block_table; /* [batch, max_blocks] */
  const int* seq_lens;    /* [batch], lengths after the append */
  const int* cu_seqlens;  /* [batch + 1], or NULL: row b is request b's one token */
  const int* positions;   /* [rows] rotation positions, or NULL: the cache positions */
  int rows;               /* rows of q, k and v (== batch when cu_seqlens is NULL) */
  int batch;
  int max_blocks;
  int num_blocks;         /* pages of the caches; ids outside [0, num_blocks) are refused */
  int block_size;         /* tokens per page */
} kv_append_tokens;

/* Rotation: table row p holds cos(p f_j) then sin(p f_j), j < rotary_dim / 2.
 * interleaved == 0 rotates the pairs (j, j + rotary_dim / 2), interleaved != 0
 * the pairs (2 j, 2 j + 1).  table NULL: no rotation. */
typedef struct kv_append_rope {
  const float* table; /* [max_positions, rotary_dim] */
  int rotary_dim;     /* a multiple of 16 up to 128 (64 for the latent cache) */
  int max_positions;
  int interleaved;
} kv_append_rope;

/* Rows of bf16 heads: element (t, h, d) at data[t * token_stride + h * head_stride + d]. */
typedef struct kv_append_heads {
  const gqa_bf16* data;
  long long token_stride;
  long long head_stride;
} kv_append_heads;

/* RMS norm weights: y = x * rsqrt(mean(x^2) + eps) * weight.  weight NULL: no norm. */
typedef struct kv_append_norm {
  const void* weight; /* bf16, or fp32 when is_fp32 != 0 */
  int is_fp32;
  float eps;
} kv_append_norm;

/* q [rows, Hq, 128] -> q_out (same strides kind), k and v [rows, Hkv, 128] ->
 * k_cache and v_cache [num_blocks, block_size, Hkv, 128].  q.data NULL: only
 * K and V.  q_out may be q itself; caches that overlap are refused.  Values
 * are held in fp32 between the load and one rounding to bf16 at the store. */
cudaError_t kv_append_gqa_launch(const kv_append_tokens* tokens, const kv_append_rope* rope,
                                 kv_append_heads q, kv_append_heads k, kv_append_heads v,
                                 kv_append_norm q_norm, kv_append_norm k_norm, gqa_bf16* q_out,
                                 long long q_out_token_stride, long long q_out_head_stride,
                                 int zero_skipped, gqa_bf16* k_cache, gqa_bf16* v_cache, int Hq,
                                 int Hkv, cudaStream_t stream);

/* kv_append_gqa_launch into the 4-bit tiles of kv4_decode.h (group 32, 64 or
 * 128; block_size a multiple of 16).  K is quantised from its fp32 value
 * after the norm and the rotation. */
cudaError_t kv_append_gqa_kv4_launch(const kv_append_tokens* tokens, const kv_append_rope* rope,
                                     kv_append_heads q, kv_append_heads k, kv_append_heads v,
                                     kv_append_norm q_norm, kv_append_norm k_norm,
                                     gqa_bf16* q_out, long long q_out_token_stride,
                                     long long q_out_head_stride, int zero_skipped,
                                     unsigned char* k_cache, unsigned char* v_cache, int Hq,
                                     int Hkv, int group, cudaStream_t stream);

/* The latent cache's append: kv_c [rows, 512] (normed) and k_pe [rows, 64]
 * (rotated) -> kv_cache [num_blocks, 64, 1, 576]; q_pe [rows, h_q, 64] ->
 * rotated q_pe_out, e.g. the last 64 dims of the decode's q.  q_pe.data NULL:
 * only the cache.  head_stride of kv_c and k_pe is not used. */
cudaError_t kv_append_mla_launch(const kv_append_tokens* tokens, const kv_append_rope* rope,
                                 kv_append_heads kv_c, kv_append_heads k_pe, kv_append_norm norm,
                                 kv_append_heads q_pe, gqa_bf16* q_pe_out,
                                 long long q_out_token_stride, long long q_out_head_stride,
                                 int zero_skipped, gqa_bf16* kv_cache, int h_q,
                                 cudaStream_t stream);

/* Status word of the append kernels on the current device: bit 1 (value 2) = a
 * block id outside [0, num_blocks): that token's K and V were not written; bit 3
 * (value 8) = a position outside the block table's row or the rotation
 * table: that row was treated as holding no token.  reset clears it.
 * Synchronises the device; negative: the read failed. */
int kv_append_get_status(int reset);

#ifdef __cplusplus
}
#endif

#endif /* KV_APPEND_B200_H */
