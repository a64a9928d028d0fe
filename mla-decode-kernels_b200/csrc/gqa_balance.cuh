// The balanced schedule's cut, shared by the decode scans.
#pragma once

#include <cuda_runtime.h>

namespace gqa {

// BALANCED ranges: the T stages of all rows, in row order, are cut into E =
// min(grid, T / 2) ranges with proportional boundaries [c T / E, (c+1) T / E)
// - sizes differ by at most one stage, and every range holds at least two
// stages so that no row is cut into single-stage parts.  CTAs c >= E idle.
__device__ __forceinline__ long long range_parts(long long T, long long grid) {
  return max(1LL, min(grid, T / 2));
}

__device__ __forceinline__ long long range_start(long long c, long long T, long long E) {
  return c >= E ? T : c * T / E;
}

// The range that holds stage g (0 <= g < T): the largest c with
// c T / E <= g, i.e. c T < (g + 1) E.
__device__ __forceinline__ long long range_owner(long long g, long long T, long long E) {
  return ((g + 1) * E - 1) / T;
}

// Block-wide start of the CTA's range in the BALANCED schedule; stages(b) =
// 16-token stages of request b, each of which has NHG rows of that length.
// Every thread takes part; afterwards sh_info holds {first stage, end, E,
// first request, stages of the requests before it, T} (sh_warp: 32 words of
// scratch).
template <class Stages>
__device__ __forceinline__ void balanced_start(int B, int NHG, Stages stages, long long* sh_warp,
                                               long long* sh_info) {
  constexpr unsigned kAll = 0xffffffffu;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nthr = blockDim.x, nwarps = nthr >> 5;
  const int chunk = (B + nthr - 1) / nthr;
  const int blo = min(B, tid * chunk), bhi = min(B, blo + chunk);
  long long local = 0;
  for (int b = blo; b < bhi; ++b) local += stages(b);
  long long x = local;
  #pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long y = __shfl_up_sync(kAll, x, off);
    if (lane >= off) x += y;
  }
  if (lane == 31) sh_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long t = lane < nwarps ? sh_warp[lane] : 0;
    #pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(kAll, t, off);
      if (lane >= off) t += y;
    }
    if (lane < nwarps) sh_warp[lane] = t;
  }
  __syncthreads();
  const long long excl = x - local + (warp > 0 ? sh_warp[warp - 1] : 0);
  const long long total = sh_warp[nwarps - 1];
  const long long T = total * NHG;
  const long long E = range_parts(T, gridDim.x);
  const long long g0 = range_start(blockIdx.x, T, E);
  const long long g1 = range_start(blockIdx.x + 1LL, T, E);
  if (tid == 0) {
    sh_info[0] = g0;
    sh_info[1] = g1;
    sh_info[2] = E;
    sh_info[3] = 0;  // first request
    sh_info[4] = 0;  // stages before it
    sh_info[5] = T;
  }
  __syncthreads();
  if (g0 < g1 && g0 >= excl * NHG && g0 < (excl + local) * NHG) {
    long long P = excl;
    for (int b = blo; b < bhi; ++b) {
      const long long L = stages(b);
      if (g0 < (P + L) * NHG) {
        sh_info[3] = b;
        sh_info[4] = P;
        break;
      }
      P += L;
    }
  }
  __syncthreads();
}

}  // namespace gqa
