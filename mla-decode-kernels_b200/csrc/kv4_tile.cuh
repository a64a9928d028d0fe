// The 4-bit cache's tile (include/kv4_decode.h): 16 tokens of one kv head.
//
// The byte order follows the decode's tensor-core fragments (m16n8k16,
// lane = 4 g + t): for K one lane needs 16 bytes of one token, its words
// 4 i + t (i = 0..3, dims 8 (4 i + t) ..), and for V^T 16 bytes of one token
// pair, dims 32 y + 4 g .. + 3 (y = 0..3) of both tokens.  Each is one
// 16-byte shared-memory load; the xor on V's chunk index spreads the four
// token pairs of a quarter warp over all banks.
#pragma once

#include <cstdint>

namespace gqa {
namespace kv4 {

constexpr int kTileTokens = 16;
constexpr int kCodeBytes = 1024;

__host__ __device__ constexpr int tile_bytes(int group) { return kCodeBytes + 64 * (128 / group); }

// Byte of K's 32-bit word w (dims 8 w ..) of token i.
__host__ __device__ constexpr int k_word(int i, int w) { return 64 * i + 16 * (w & 3) + 4 * (w >> 2); }

// Byte of V's 16 bits of dims 4 r .. 4 r + 3 of token i.
__host__ __device__ constexpr int v_half(int i, int r) {
  return 128 * (i >> 1) + 16 * ((r & 7) ^ (2 * ((i >> 1) & 3))) + 4 * (r >> 3) + 2 * (i & 1);
}

// Bytes of the scale and the centre of token i, dim group y of ng.
__host__ __device__ constexpr int scale_at(int i, int y, int ng) {
  return kCodeBytes + 2 * (ng * i + y);
}
__host__ __device__ constexpr int k_centre_at(int i, int y, int ng) {
  return kCodeBytes + 32 * ng + 2 * (ng * i + y);
}
__host__ __device__ constexpr int v_centre_at(int i, int y, int ng) {
  return kCodeBytes + 32 * ng + 2 * (16 * y + i);
}

}  // namespace kv4
}  // namespace gqa
