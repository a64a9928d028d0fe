/*
 * GQA decode over a paged cache held in 4 bits, C ABI.
 *
 * The operator is gqa_decode.h's, with K and V stored as 4-bit codes: the
 * `group` (32, 64 or 128) consecutive dims of one token and kv head share a
 * bf16 scale s and a bf16 centre c, and code n stands for s * (n - 8) + c.
 * Scales are not negative.
 * The quantiser (kv_append_gqa_kv4_launch) takes, over the group's fp32
 * values x, s = (max - min) / 15 rounded up to bf16, c = min + 8 s rounded
 * to nearest bf16 and n = clamp(round((x - c) / s) + 8, 0, 15) (n = 8 where
 * s = 0).  No code is clipped but for c's rounding to bf16, which shifts
 * a group's codes where |c| is large against its range (mean 20, deviation
 * 0.3: errors of up to a step; mean 100: three).  A group that holds a NaN or
 * an infinity, or whose range passes fp32's, reads back as NaN; in the decode
 * it spoils all dims of the request's q heads of its kv head.
 *
 * K and V caches are uint8 [num_blocks, block_size / 16, Hkv, tile], tile =
 * 1024 + 64 * (128 / group) bytes: one tile is 16 tokens of one kv head,
 * arranged so that the decode's tensor-core fragments are 16-byte pieces of
 * it without bank conflicts.  ng = 128 / group:
 *   K codes  token i's 64 bytes at 64 i; the 32-bit word of dims 8 w .. 8 w + 7
 *            (nibble j = dim 8 w + j) at byte 16 (w % 4) + 4 (w / 4) of them;
 *   V codes  tokens 2 p and 2 p + 1 at 128 p; the 16 bits of dims 4 r .. 4 r + 3,
 *            r = 8 y + g, of token 2 p + e at byte 16 (g ^ 2 (p % 4)) + 4 y + 2 e;
 *   scales   bf16 [16][ng] at 1024;
 *   centres  bf16 at 1024 + 32 ng: K [16][ng], V [ng][16].
 * Bytes per cached value: 0.5 + 4 / group (K1's bf16 cache: 2).
 *
 * The reference has no counterpart.  Every launcher is asynchronous on
 * `stream`, allocates nothing and does not synchronise.
 */
#ifndef KV4_DECODE_B200_H
#define KV4_DECODE_B200_H

#include <stddef.h>
#include <cuda_runtime_api.h>

#include "gqa_decode.h" /* gqa_bf16 */

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one tile, 0 for a group that is not 32, 64 or 128. */
size_t kv4_tile_bytes(int group);

/* Workspace bytes of kv4_decode_launch on the current device (no
 * initialisation needed); 0 for invalid dims. */
size_t kv4_decode_workspace_bytes(int B, int Hq, int Hkv, int group);

/* out[b, h] = softmax_t(q[b, h] . K[t] * scale) @ V[t] over t < seq_lens[b]
 * (0 for a request without tokens); q and out bf16 [B, Hq, 128], block_table
 * int32 [B, max_blocks], seq_lens int32 [B], lengths past the block table's
 * row count as its end and negative ones as 0.  block_size a multiple of 16,
 * q, out, caches and workspace 16-byte aligned.  A block id outside
 * [0, num_blocks) sets bit 1 of kv4_decode_get_status and reads block 0.
 * Calls that may overlap on the GPU must not share a workspace. */
cudaError_t kv4_decode_launch(const gqa_bf16* q, const unsigned char* k_cache,
                              const unsigned char* v_cache, const int* block_table,
                              const int* seq_lens, gqa_bf16* out, int B, int Hq, int Hkv,
                              int group, int block_size, int max_blocks, int num_blocks,
                              float scale, void* workspace, size_t workspace_bytes,
                              cudaStream_t stream);

/* Read tokens back as bf16, e.g. for a prompt's attention over a cached
 * prefix: the last cu_seqlens[b + 1] - cu_seqlens[b] of request b's
 * seq_lens[b] tokens into rows cu_seqlens[b] .. of k and v [rows, Hkv, 128]
 * (cu_seqlens NULL: its last token into row b).  Rows that hold no token are
 * zero.  Block ids outside [0, num_blocks) set bit 1 of the status and read
 * block 0; a position past the block table's row sets bit 3 and reads zero. */
cudaError_t kv4_gather_launch(const unsigned char* k_cache, const unsigned char* v_cache,
                              const int* block_table, const int* seq_lens, const int* cu_seqlens,
                              gqa_bf16* k, gqa_bf16* v, int rows, int B, int Hkv, int group,
                              int block_size, int max_blocks, int num_blocks,
                              cudaStream_t stream);

/* Status word of the 4-bit cache's kernels on the current device (bit 0: a
 * bounded wait gave up, bit 1: block id out of range, bit 3: position out of
 * range); reset clears it.  Synchronises the device; negative: the read failed. */
int kv4_decode_get_status(int reset);

#ifdef __cplusplus
}
#endif

#endif /* KV4_DECODE_B200_H */
