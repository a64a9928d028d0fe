// Where the rows of a ragged batch of tokens lie in the paged cache, shared
// by the append kernels and the 4-bit cache's read-back.
#pragma once

#include <cstdint>

#include "launch_early.cuh"

namespace gqa {

constexpr int kStatusBadPosition = 8;  // position past the table's row or the rotation table

struct Tokens {
  const int* block_table;  // [batch, max_blocks]
  const int* seq_lens;     // [batch], lengths with the rows included
  const int* cu;           // [batch + 1] rows of every request, or null: one row each
  const int* positions;    // [rows] rotation positions, or null
  int rows, batch, max_blocks, num_blocks, block_size;
};

struct Place {
  int b, pos;     // request and cache position
  int rope_pos;   // rotation position
  bool live;      // the row holds a token
};

// The number of i in [1, batch] with cu[i] <= t, found by the whole warp: 32
// samples per step, so a batch of up to 32 takes one load and one of up to
// 1024 two.  cu must not decrease; other contents give some value in
// [0, batch].
__device__ __forceinline__ int find_request(const int* cu, int batch, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = batch;  // the answer is in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int i = lo + (lane + 1) * step;  // sample: is cu[i] <= t?
    const bool in = (lane + 1) * step <= n;
    const bool le = in && ld_plain(cu + i) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));  // samples passed
    lo += c * step;
    n = min(n - c * step, step - 1);
  }
  return lo;
}

// The place of row t; every lane of the warp must call it with the same t.
__device__ __forceinline__ Place find_place(const Tokens& k, int t) {
  Place p{t, 0, 0, false};
  int end = t + 1;  // rows of the request end here
  if (k.cu) {
    p.b = find_request(k.cu, k.batch, t);
    if (p.b >= k.batch || t < ld_plain(k.cu + p.b)) return p;
    end = ld_plain(k.cu + p.b + 1);
  } else if (t >= k.batch) {
    return p;
  }
  p.pos = ld_plain(k.seq_lens + p.b) - (end - t);
  p.live = p.pos >= 0;
  p.rope_pos = k.positions ? ld_plain(k.positions + t) : p.pos;
  return p;
}

}  // namespace gqa
