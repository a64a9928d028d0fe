// GQA decode over the 4-bit paged cache (include/kv4_decode.h), and the
// read-back of cached tokens as bf16.
//
// Mathematics.  Code n of K or V stands for s (n - 8) + c, s and c shared by
// the `group` dims y of a token.  With Q_y = sum of q over group y,
//     q . k_t = sum_y s_ty (sum_d q_d (n_td - 8)) + sum_y c_ty Q_y,
//     out_d   = sum_t (p_t s_ty) (n_td - 8) + sum_t p_t c_ty,
// so neither scale nor centre is ever applied to a code: K's products with
// the raw codes are summed per group on the tensor cores and scaled after,
// V's scales are folded into the softmax weights of each group, and both
// centre terms are one small tensor-core product per tile.  A code becomes
// bf16 128 + n by one and-or on its word; K removes the offset through the
// accumulator's start value -136 Q_y, V by one packed subtraction (exact),
// since over a long sequence the sum of 136 p s would swamp fp32.
//
// CTA layout (one persistent CTA per SM, the balanced schedule of
// gqa_balance.cuh, cut rows merged by the cut-row merge kernel):
//   * the last warp copies tiles (cp.async.bulk, one per 16-token tile and
//     row of HG kv heads: contiguous in the cache) into a ring whose slots
//     hold K or V of 2 TS tiles;
//   * HG x NT x TS consumer warps: kv head, 8 of its q heads, and every
//     TS-th pair of tiles.  The TS warps of a head keep their own softmax
//     state and meet in shared memory at the end of a segment.
#include <math.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "device_once.h"
#include "gqa_balance.cuh"
#include "gqa_internal.h"
#include "gqa_ptx.cuh"
#include "kv4_decode.h"
#include "kv4_tile.cuh"
#include "kv_tokens.cuh"

namespace gqa {
namespace kv4 {

__device__ int g_kv4_status;

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxWarps = 16;                // consumer warps
constexpr int kMaxSlots = 16;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kStateWords = 36;              // floats per lane of a warp's softmax state
constexpr int kStateBytes = kStateWords * 32 * 4;

__device__ __forceinline__ void raise_status(int bits) { atomicOr(&g_kv4_status, bits); }

// How a launch maps to warps and shared memory (no device state).
struct Plan {
  int G, NT, HG, NHG, TS, ncw;
  int slot_tiles, slot_bytes, nslots, smem;
};

struct DecodeParams {
  const __nv_bfloat16* q;
  const unsigned char* k;
  const unsigned char* v;
  const int* block_table;
  const int* seq_lens;
  __nv_bfloat16* out;
  float* part_m;
  float* part_l;
  float* part_acc;
  int2* row_info;
  int2* ends;
  int B, Hq, Hkv, tiles_per_block, max_blocks, num_blocks;
  float scale_log2;
  Plan pl;
};

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes j and j + 4 of a word as the bf16 pair (128 + n, 128 + n'): exact,
// bf16 has 7 fraction bits and 128's last one stands for 1.
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int j) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(w >> (4 * j)));  // (a & b) | c
  return r;
}

// (128 + n) - 136 = n - 8, exact in bf16.
__device__ __forceinline__ uint32_t centred(uint32_t pair) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pair), "r"(0x43084308u));
  return r;
}

// The NG bf16 scales of one token as floats.
template <int NG>
__device__ __forceinline__ void load_scales(uint32_t a, float (&s)[NG]) {
  if constexpr (NG == 4) {
    uint32_t x, y;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(a));
    s[0] = __uint_as_float(x << 16);
    s[1] = __uint_as_float(x & 0xffff0000u);
    s[2] = __uint_as_float(y << 16);
    s[3] = __uint_as_float(y & 0xffff0000u);
  } else if constexpr (NG == 2) {
    const uint32_t x = lds32(a);
    s[0] = __uint_as_float(x << 16);
    s[1] = __uint_as_float(x & 0xffff0000u);
  } else {
    s[0] = __uint_as_float(lds16(a) << 16);
  }
}

struct Seg {
  int b, hg, row, S, s0, s1, nparts, slot;
  long long cfirst;
};

// The CTA's share of the balanced schedule, as segments (one row, a range of
// its tiles).
struct Walk {
  long long g, g_end, T, E, row0;
  int b, hg, S, L;
};

__device__ __forceinline__ int req_len(const DecodeParams& p, int b) {
  const int s = ld_nc_s32(p.seq_lens + b);
  const long long cap = static_cast<long long>(p.max_blocks) * p.tiles_per_block * kTileTokens;
  return s < 0 ? 0 : static_cast<int>(min(static_cast<long long>(s), cap));
}

__device__ __forceinline__ int req_tiles(const DecodeParams& p, int b) {
  return static_cast<int>((static_cast<long long>(req_len(p, b)) + kTileTokens - 1) / kTileTokens);
}

__device__ __forceinline__ bool next_seg(Walk& w, const DecodeParams& p, Seg& s) {
  while (w.g < w.g_end) {
    const long long rs = w.row0 + static_cast<long long>(w.hg) * w.L, re = rs + w.L;
    if (w.g >= re) {
      if (++w.hg == p.pl.NHG) {
        w.hg = 0;
        w.row0 += static_cast<long long>(p.pl.NHG) * w.L;
        if (++w.b >= p.B) {
          w.g = w.g_end;
          return false;
        }
        w.S = req_len(p, w.b);
        w.L = req_tiles(p, w.b);
      }
      continue;
    }
    const long long e = min(w.g_end, re);
    s.b = w.b;
    s.hg = w.hg;
    s.row = w.b * p.pl.NHG + w.hg;
    s.S = w.S;
    s.s0 = static_cast<int>(w.g - rs);
    s.s1 = static_cast<int>(e - rs);
    s.cfirst = range_owner(rs, w.T, w.E);
    s.nparts = static_cast<int>(range_owner(re - 1, w.T, w.E) - s.cfirst + 1);
    s.slot = static_cast<int>(blockIdx.x) + s.row;
    w.g = e;
    return true;
  }
  return false;
}

__device__ __forceinline__ void group_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// A warp's softmax state: lane (g, t) holds heads 2 t and 2 t + 1 (n = 0, 1),
// dims 32 y + 4 g + 2 u + v in acc[2 y + u][2 v + n].
struct State {
  float m[2], l[2];
  float acc[8][4];
};

__device__ __forceinline__ void merge_state(State& a, const float* other, int lane) {
  #pragma unroll
  for (int n = 0; n < 2; ++n) {
    const float mo = other[n * 32 + lane], lo = other[(2 + n) * 32 + lane];
    const float m = fmaxf(a.m[n], mo);
    const float fa = a.m[n] == -INFINITY ? 0.f : exp2_approx(a.m[n] - m);
    const float fo = mo == -INFINITY ? 0.f : exp2_approx(mo - m);
    a.m[n] = m;
    a.l[n] = a.l[n] * fa + lo * fo;
    #pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      a.acc[mt][n] = a.acc[mt][n] * fa + other[(4 + 4 * mt + n) * 32 + lane] * fo;
      a.acc[mt][2 + n] = a.acc[mt][2 + n] * fa + other[(4 + 4 * mt + 2 + n) * 32 + lane] * fo;
    }
  }
}

__device__ __forceinline__ void put_state(const State& a, float* dst, int lane) {
  #pragma unroll
  for (int n = 0; n < 2; ++n) {
    dst[n * 32 + lane] = a.m[n];
    dst[(2 + n) * 32 + lane] = a.l[n];
  }
  #pragma unroll
  for (int mt = 0; mt < 8; ++mt)
    #pragma unroll
    for (int i = 0; i < 4; ++i) dst[(4 + 4 * mt + i) * 32 + lane] = a.acc[mt][i];
}

}  // namespace

template <int NG>
__global__ void __launch_bounds__((kMaxWarps + 1) * 32, 1)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kGroup = 128 / NG, kTile = tile_bytes(kGroup);
  constexpr float kThreshold = 8.f;  // log2 units a score may pass the running maximum by
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long sh_warp[32];
  __shared__ long long sh_info[8];
  __shared__ __align__(8) unsigned long long sh_bar[2 * kMaxSlots];

  const Plan& pl = p.pl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem);
  const uint32_t full = smem_u32(sh_bar), empty = full + 8u * kMaxSlots;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < pl.nslots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, pl.ncw);
    }
    fence_mbar_init();
  }
  balanced_start(
      p.B, pl.NHG, [&](int b) -> long long { return req_tiles(p, b); }, sh_warp, sh_info);

  Walk walk;
  walk.g = sh_info[0];
  walk.g_end = sh_info[1];
  walk.E = sh_info[2];
  walk.b = static_cast<int>(sh_info[3]);
  walk.row0 = sh_info[4] * pl.NHG;
  walk.T = sh_info[5];
  walk.hg = 0;
  walk.S = walk.g < walk.g_end ? req_len(p, walk.b) : 0;
  walk.L = (walk.S + kTileTokens - 1) / kTileTokens;
  Seg s;

  if (warp == pl.ncw) {
    // ------------------------------ producer ------------------------------
    const uint64_t pol = policy_evict_first();
    const uint32_t row_bytes = static_cast<uint32_t>(pl.HG * kTile);
    int slot = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    while (ok && next_seg(walk, p, s)) {
      const int* table = p.block_table + static_cast<size_t>(s.b) * p.max_blocks;
      for (int st = s.s0; st < s.s1 && ok; st += pl.slot_tiles) {
        const int nt = min(pl.slot_tiles, s.s1 - st);
        size_t off = 0;
        if (lane < nt) {
          const int tile = st + lane;
          const int lb = tile / p.tiles_per_block, sub = tile - lb * p.tiles_per_block;
          int page = __ldg(table + lb);
          if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
            raise_status(kStatusBadPage);
            page = 0;
          }
          off = ((static_cast<size_t>(page) * p.tiles_per_block + sub) * p.Hkv +
                 static_cast<size_t>(s.hg) * pl.HG) * kTile;
        }
        #pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!__all_sync(kFull, mbar_wait(empty + 8 * slot, phase ^ 1))) {
            raise_status(kStatusWaitTimeout);
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(full + 8 * slot, row_bytes * nt);
          __syncwarp();
          if (lane < nt)
            bulk_g2s(ring + slot * pl.slot_bytes + lane * row_bytes, (kv ? p.v : p.k) + off,
                     row_bytes, full + 8 * slot, pol);
          ++issued;
          if (++slot == pl.nslots) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
    }
    // No copy may land after the CTA has exited (see the K1 scan).
    const long long inflight = min(issued, static_cast<long long>(pl.nslots));
    for (long long j = 1; j <= inflight; ++j) {
      const long long idx = issued - j;
      mbar_wait(full + 8 * static_cast<int>(idx % pl.nslots),
                static_cast<uint32_t>((idx / pl.nslots) & 1));
    }
    return;
  }

  // ------------------------------ consumers -------------------------------
  const int team = warp / pl.TS, ts = warp - team * pl.TS;  // team = (kv head, q-head tile)
  const int hl = team / pl.NT, j0 = (team - hl * pl.NT) * 8;
  const int cnt = min(8, pl.G - j0);
  const int g = lane >> 2, t = lane & 3;
  float* scratch = reinterpret_cast<float*>(smem + pl.nslots * pl.slot_bytes) +
                   static_cast<size_t>(team) * (pl.TS / 2) * (kStateBytes / 4);

  // Requests without tokens occupy no tiles: CTA (b mod grid) zeroes them.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (req_len(p, b) != 0) continue;
    if (ts == 0)
      for (int hg = 0; hg < pl.NHG; ++hg)
        for (int n = 0; n < cnt; ++n)
          *reinterpret_cast<uint2*>(
              p.out + (static_cast<size_t>(b) * p.Hq + (hg * pl.HG + hl) * pl.G + j0 + n) * kHeadDim +
              4 * lane) = make_uint2(0, 0);
  }
  if (warp == 0 && lane == 0) p.ends[blockIdx.x] = make_int2(-1, 0);

  int slot = 0;
  uint32_t phase = 0;
  bool dead = false;  // a wait gave up: empty states from here on (see the K1 scan)
  bool first_seg = true;
  const auto advance = [&]() {
    if (++slot == pl.nslots) {
      slot = 0;
      phase ^= 1;
    }
  };

  while (next_seg(walk, p, s)) {
    const int hbase = (s.hg * pl.HG + hl) * pl.G + j0;
    if (warp == 0 && lane == 0) {
      if (first_seg && s.nparts > 1 && s.s1 == (s.S + kTileTokens - 1) / kTileTokens)
        p.ends[blockIdx.x] = make_int2(s.row, s.nparts);
      if (s.s0 == 0) p.row_info[s.row] = make_int2(static_cast<int>(s.cfirst), s.nparts);
    }
    first_seg = false;

    // q fragments (B operand): lane (g, t) holds head g, words 4 i + t.
    uint32_t qf[8][2];
    uint32_t qsum_b;        // group sums of q, high and low bf16 parts, as a B operand
    float start[NG][2];     // -136 Q of heads 2 t, 2 t + 1
    {
      const bool has = g < cnt;
      const __nv_bfloat16* qrow =
          p.q + (static_cast<size_t>(s.b) * p.Hq + hbase + (has ? g : 0)) * kHeadDim;
      float qs[4];
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 w = has ? __ldg(reinterpret_cast<const uint4*>(qrow + 8 * (4 * i + t)))
                            : make_uint4(0, 0, 0, 0);
        // dims (0, 4), (1, 5), (2, 6), (3, 7) of the word
        qf[2 * i][0] = __byte_perm(w.x, w.z, 0x5410);
        qf[2 * i][1] = __byte_perm(w.x, w.z, 0x7632);
        qf[2 * i + 1][0] = __byte_perm(w.y, w.w, 0x5410);
        qf[2 * i + 1][1] = __byte_perm(w.y, w.w, 0x7632);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        float a = 0.f;
        #pragma unroll
        for (int k = 0; k < 4; ++k)
          a += __uint_as_float(u[k] << 16) + __uint_as_float(u[k] & 0xffff0000u);
        a += __shfl_xor_sync(kFull, a, 1);
        a += __shfl_xor_sync(kFull, a, 2);
        qs[i] = a;
      }
      float Q[NG];
      #pragma unroll
      for (int y = 0; y < NG; ++y) {
        Q[y] = 0.f;
        #pragma unroll
        for (int i = 0; i < 4 / NG; ++i) Q[y] += qs[y * (4 / NG) + i];
        start[y][0] = -136.f * __shfl_sync(kFull, Q[y], 8 * t);
        start[y][1] = -136.f * __shfl_sync(kFull, Q[y], 8 * t + 4);
      }
      float hi[NG], lo[NG];
      #pragma unroll
      for (int y = 0; y < NG; ++y) {
        hi[y] = __bfloat162float(__float2bfloat16(Q[y]));
        lo[y] = Q[y] - hi[y];
      }
      if constexpr (NG == 4) {
        const uint32_t h01 = pack_bf16x2(hi[0], hi[1]), h23 = pack_bf16x2(hi[2], hi[3]);
        const uint32_t l01 = pack_bf16x2(lo[0], lo[1]), l23 = pack_bf16x2(lo[2], lo[3]);
        qsum_b = t < 2 ? (t == 0 ? h01 : h23) : (t == 2 ? l01 : l23);
      } else if constexpr (NG == 2) {
        qsum_b = t == 0 ? pack_bf16x2(hi[0], hi[1]) : (t == 1 ? pack_bf16x2(lo[0], lo[1]) : 0u);
      } else {
        qsum_b = t == 0 ? pack_bf16x2(hi[0], lo[0]) : 0u;
      }
    }

    State a;
    a.m[0] = a.m[1] = -INFINITY;
    a.l[0] = a.l[1] = 0.f;
    #pragma unroll
    for (int mt = 0; mt < 8; ++mt) a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;
    float cw[4] = {0.f, 0.f, 0.f, 0.f};  // sum_t p_t c_ty: row y = g, heads 2 t, 2 t + 1

    for (int st = s.s0; st < s.s1 && !dead; st += pl.slot_tiles) {
      const int mine = min(2, min(pl.slot_tiles, s.s1 - st) - 2 * ts);  // tiles of this warp
      const uint32_t tile0 = static_cast<uint32_t>((2 * ts * pl.HG + hl) * kTile);
      const uint32_t tile_step = static_cast<uint32_t>(pl.HG * kTile);
      const int left = s.S - (st + 2 * ts) * kTileTokens;  // valid tokens from tile 0 on
      float x[2][4];

      if (!__all_sync(kFull, mbar_wait(full + 8 * slot, phase))) {
        dead = true;
        break;
      }
      if (mine > 0) {
        const uint32_t kb = ring + slot * pl.slot_bytes + tile0;
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[j][0] = x[j][1] = x[j][2] = x[j][3] = -INFINITY;
          if (j < mine) {
            const uint32_t tb = kb + j * tile_step;
            const uint4 wa = lds128(tb + 64 * g + 16 * t), wb = lds128(tb + 512 + 64 * g + 16 * t);
            const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
            float sa[NG], sb[NG];
            load_scales<NG>(tb + scale_at(0, 0, NG) + 2 * NG * g, sa);
            load_scales<NG>(tb + scale_at(8, 0, NG) + 2 * NG * g, sb);
            uint32_t ca, cb;
            if constexpr (NG == 4) {
              ca = lds32(tb + k_centre_at(0, 0, NG) + 8 * g + 4 * (t & 1));
              cb = lds32(tb + k_centre_at(8, 0, NG) + 8 * g + 4 * (t & 1));
            } else if constexpr (NG == 2) {
              ca = lds32(tb + k_centre_at(0, 0, NG) + 4 * g);
              cb = lds32(tb + k_centre_at(8, 0, NG) + 4 * g);
            } else {
              ca = lds16(tb + k_centre_at(0, 0, NG) + 2 * g) * 0x10001u;
              cb = lds16(tb + k_centre_at(8, 0, NG) + 2 * g) * 0x10001u;
            }
            float sc[4] = {0.f, 0.f, 0.f, 0.f};
            mma_bf16_16816(sc, ca, cb, 0u, 0u, qsum_b, 0u);
            #pragma unroll
            for (int y = 0; y < NG; ++y) {
              float d[4] = {start[y][0], start[y][1], start[y][0], start[y][1]};
              #pragma unroll
              for (int i = y * (4 / NG); i < (y + 1) * (4 / NG); ++i) {
                mma_bf16_16816(d, code_pair(ua[i], 0), code_pair(ub[i], 0), code_pair(ua[i], 1),
                               code_pair(ub[i], 1), qf[2 * i][0], qf[2 * i][1]);
                mma_bf16_16816(d, code_pair(ua[i], 2), code_pair(ub[i], 2), code_pair(ua[i], 3),
                               code_pair(ub[i], 3), qf[2 * i + 1][0], qf[2 * i + 1][1]);
              }
              sc[0] += sa[y] * d[0];
              sc[1] += sa[y] * d[1];
              sc[2] += sb[y] * d[2];
              sc[3] += sb[y] * d[3];
            }
            const int nv = left - j * kTileTokens;
            x[j][0] = g < nv ? sc[0] * p.scale_log2 : -INFINITY;
            x[j][1] = g < nv ? sc[1] * p.scale_log2 : -INFINITY;
            x[j][2] = g + 8 < nv ? sc[2] * p.scale_log2 : -INFINITY;
            x[j][3] = g + 8 < nv ? sc[3] * p.scale_log2 : -INFINITY;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * slot);
      advance();

      if (mine > 0) {
        float mx[2];
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
          mx[n] = fmaxf(fmaxf(x[0][n], x[0][2 + n]), fmaxf(x[1][n], x[1][2 + n]));
          #pragma unroll
          for (int off = 4; off < 32; off <<= 1)
            mx[n] = fmaxf(mx[n], __shfl_xor_sync(kFull, mx[n], off));
        }
        // The running maximum moves only when a score passes it by more than
        // kThreshold: weights stay below 2^8 and most tiles rescale nothing.
        if (__any_sync(kFull, mx[0] > a.m[0] + kThreshold || mx[1] > a.m[1] + kThreshold)) {
          #pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float m = fmaxf(a.m[n], mx[n]);
            const float f = a.m[n] == -INFINITY ? 0.f : exp2_approx(a.m[n] - m);
            a.m[n] = m;
            a.l[n] *= f;
            cw[n] *= f;
            #pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
              a.acc[mt][n] *= f;
              a.acc[mt][2 + n] *= f;
            }
          }
        }
        #pragma unroll
        for (int j = 0; j < 2; ++j)
          #pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[j][i] = exp2_approx(x[j][i] - a.m[i & 1]);
            a.l[i & 1] += x[j][i];
          }
      }

      if (!__all_sync(kFull, mbar_wait(full + 8 * slot, phase))) {
        dead = true;
        break;
      }
      if (mine > 0) {
        const uint32_t vb = ring + slot * pl.slot_bytes + tile0;
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j < mine) {
            const uint32_t tb = vb + j * tile_step;
            const uint32_t va = tb + 128 * t + 16 * (g ^ (2 * t));
            const uint4 wa = lds128(va), wb = lds128(va + 512);
            const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
            float sa[NG], sb[NG];
            load_scales<NG>(tb + scale_at(0, 0, NG) + 2 * NG * g, sa);
            load_scales<NG>(tb + scale_at(8, 0, NG) + 2 * NG * g, sb);
            uint32_t ca = 0u, cb = 0u;
            if (g < NG) {
              ca = lds32(tb + v_centre_at(0, 0, NG) + 32 * g + 4 * t);
              cb = lds32(tb + v_centre_at(8, 0, NG) + 32 * g + 4 * t);
            }
            const int nv = left - j * kTileTokens;
            if (nv < kTileTokens) {
              // what lies behind the last token may be anything: no scale, no centre
              #pragma unroll
              for (int y = 0; y < NG; ++y) {
                if (g >= nv) sa[y] = 0.f;
                if (g + 8 >= nv) sb[y] = 0.f;
              }
              if (2 * t >= nv) ca = 0u; else if (2 * t + 1 >= nv) ca &= 0xffffu;
              if (2 * t + 8 >= nv) cb = 0u; else if (2 * t + 9 >= nv) cb &= 0xffffu;
            }
            mma_bf16_16816(cw, ca, 0u, cb, 0u, movmatrix_trans(pack_bf16x2(x[j][0], x[j][1])),
                           movmatrix_trans(pack_bf16x2(x[j][2], x[j][3])));
            #pragma unroll
            for (int y = 0; y < NG; ++y) {
              const uint32_t b0 = movmatrix_trans(pack_bf16x2(x[j][0] * sa[y], x[j][1] * sa[y]));
              const uint32_t b1 = movmatrix_trans(pack_bf16x2(x[j][2] * sb[y], x[j][3] * sb[y]));
              #pragma unroll
              for (int i = y * (4 / NG); i < (y + 1) * (4 / NG); ++i)
                #pragma unroll
                for (int u = 0; u < 2; ++u)
                  mma_bf16_16816(a.acc[2 * i + u], centred(code_pair(ua[i], 2 * u)),
                                 centred(code_pair(ua[i], 2 * u + 1)),
                                 centred(code_pair(ub[i], 2 * u)),
                                 centred(code_pair(ub[i], 2 * u + 1)), b0, b1);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * slot);
      advance();
    }

    // ---- segment epilogue ----
    if (dead) {
      if (lane == 0) raise_status(kStatusWaitTimeout);
      a.m[0] = a.m[1] = -INFINITY;
      a.l[0] = a.l[1] = 0.f;
      cw[0] = cw[1] = 0.f;
      #pragma unroll
      for (int mt = 0; mt < 8; ++mt)
        a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;
    }
    // Teams whose segment fits in one warp's tiles skip the meeting.
    const int active = min(pl.TS, (min(pl.slot_tiles, s.s1 - s.s0) + 1) / 2);
    if (ts < active) {
      #pragma unroll
      for (int n = 0; n < 2; ++n) {
        #pragma unroll
        for (int off = 4; off < 32; off <<= 1) a.l[n] += __shfl_xor_sync(kFull, a.l[n], off);
        #pragma unroll
        for (int y = 0; y < NG; ++y) {
          const float c = __shfl_sync(kFull, cw[n], 4 * y + t);
          #pragma unroll
          for (int i = y * (4 / NG); i < (y + 1) * (4 / NG); ++i)
            #pragma unroll
            for (int u = 0; u < 2; ++u) {
              a.acc[2 * i + u][n] += c;
              a.acc[2 * i + u][2 + n] += c;
            }
        }
      }
    }
    if (active > 1) {
      for (int off = pl.TS / 2; off >= 1; off >>= 1) {
        if (off >= active) continue;  // uniform over the team
        if (ts >= off && ts < 2 * off && ts < active)
          put_state(a, scratch + (ts - off) * (kStateBytes / 4), lane);
        group_barrier(1 + team, 32 * pl.TS);
        if (ts < off && ts + off < active)
          merge_state(a, scratch + ts * (kStateBytes / 4), lane);
        group_barrier(1 + team, 32 * pl.TS);
      }
    }
    if (ts != 0) continue;
    #pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int head = 2 * t + n;
      if (head >= cnt) continue;
      if (s.nparts == 1) {
        __nv_bfloat16* o = p.out + (static_cast<size_t>(s.b) * p.Hq + hbase + head) * kHeadDim + 4 * g;
        const float inv = 1.f / a.l[n];
        #pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<uint2*>(o + 32 * y) =
              make_uint2(pack_bf16x2(a.acc[2 * y][n] * inv, a.acc[2 * y][2 + n] * inv),
                         pack_bf16x2(a.acc[2 * y + 1][n] * inv, a.acc[2 * y + 1][2 + n] * inv));
      } else {
        const size_t idx = static_cast<size_t>(s.slot) * (pl.HG * pl.G) + hl * pl.G + j0 + head;
        if (g == 0) {
          p.part_m[idx] = a.m[n];
          p.part_l[idx] = a.l[n];
        }
        float* o = p.part_acc + idx * kHeadDim + 4 * g;
        #pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<float4*>(o + 32 * y) =
              make_float4(a.acc[2 * y][n], a.acc[2 * y][2 + n], a.acc[2 * y + 1][n],
                          a.acc[2 * y + 1][2 + n]);
      }
    }
  }
}

// Read-back: half a warp per token and kv head, 8 dims per lane, K then V.
template <int NG>
__global__ void __launch_bounds__(256)
    kv4_gather_kernel(Tokens tk, const unsigned char* kc, const unsigned char* vc,
                      __nv_bfloat16* k, __nv_bfloat16* v, int Hkv) {
  constexpr int kTile = tile_bytes(128 / NG);
  const int lane = threadIdx.x & 31, l = lane & 15;
  const int per = (Hkv + 1) / 2;  // warps per token
  const long long w = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (w >= static_cast<long long>(tk.rows) * per) return;
  const int t = static_cast<int>(w / per);
  const int h = 2 * static_cast<int>(w - static_cast<long long>(t) * per) + (lane >> 4);
  Place pl = find_place(tk, t);
  const unsigned char* src_k = nullptr;
  const unsigned char* src_v = nullptr;
  int ti = 0;
  if (pl.live) {
    if (pl.pos >= static_cast<long long>(tk.max_blocks) * tk.block_size) {
      if (lane == 0) raise_status(kStatusBadPosition);
      pl.live = false;
    } else {
      const int lb = pl.pos / tk.block_size, slot = pl.pos - lb * tk.block_size;
      int page = __ldg(tk.block_table + static_cast<size_t>(pl.b) * tk.max_blocks + lb);
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(tk.num_blocks)) {
        if (lane == 0) raise_status(kStatusBadPage);
        page = 0;
      }
      ti = slot % kTileTokens;
      const size_t off = ((static_cast<size_t>(page) * (tk.block_size / kTileTokens) +
                           slot / kTileTokens) * Hkv + h) * kTile;
      src_k = kc + off;
      src_v = vc + off;
    }
  }
  if (h >= Hkv) return;
  uint4 ok = make_uint4(0, 0, 0, 0), ov = ok;
  if (pl.live) {
    const int y = 8 * l * NG / 128;
    const auto half = [](const unsigned char* a) {
      return __uint_as_float(
          static_cast<unsigned>(__ldg(reinterpret_cast<const unsigned short*>(a))) << 16);
    };
    const unsigned ck = __ldg(reinterpret_cast<const unsigned*>(src_k + k_word(ti, l)));
    const unsigned cv =
        __ldg(reinterpret_cast<const unsigned short*>(src_v + v_half(ti, 2 * l))) |
        static_cast<unsigned>(
            __ldg(reinterpret_cast<const unsigned short*>(src_v + v_half(ti, 2 * l + 1)))) << 16;
    const float sk = half(src_k + scale_at(ti, y, NG)), zk = half(src_k + k_centre_at(ti, y, NG));
    const float sv = half(src_v + scale_at(ti, y, NG)), zv = half(src_v + v_centre_at(ti, y, NG));
    const auto value = [](unsigned w, int i, float sc, float c) {
      return __fadd_rn(__fmul_rn(static_cast<float>(static_cast<int>((w >> (4 * i)) & 15u) - 8), sc), c);
    };
    unsigned a[4], b[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = pack_bf16x2(value(ck, 2 * i, sk, zk), value(ck, 2 * i + 1, sk, zk));
      b[i] = pack_bf16x2(value(cv, 2 * i, sv, zv), value(cv, 2 * i + 1, sv, zv));
    }
    ok = make_uint4(a[0], a[1], a[2], a[3]);
    ov = make_uint4(b[0], b[1], b[2], b[3]);
  }
  const size_t at = (static_cast<size_t>(t) * Hkv + h) * 128 + 8 * l;
  *reinterpret_cast<uint4*>(k + at) = ok;
  *reinterpret_cast<uint4*>(v + at) = ov;
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool valid_group(int group) { return group == 32 || group == 64 || group == 128; }

// 0, or -1 for dims the kernel does not take.
int make_plan(int Hq, int Hkv, int group, Plan* p) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || !valid_group(group)) return -1;
  p->G = Hq / Hkv;
  p->NT = (p->G + 7) / 8;
  if (p->NT > kMaxWarps) return -1;
  // kv heads per row: up to 8 warps' worth, so that two warps can share each
  // head's tokens; then as many warps per head as 16 allow.
  p->HG = 1;
  for (int d = 1; d <= Hkv && d * p->NT <= 8; ++d)
    if (Hkv % d == 0) p->HG = d;
  p->NHG = Hkv / p->HG;
  p->TS = 1;
  while (2 * p->TS * p->HG * p->NT <= kMaxWarps) p->TS *= 2;
  p->ncw = p->HG * p->NT * p->TS;
  p->slot_tiles = 2 * p->TS;
  p->slot_bytes = p->slot_tiles * p->HG * tile_bytes(group);
  const int scratch = p->HG * p->NT * (p->TS / 2) * kStateBytes;
  p->nslots = std::min(kMaxSlots, (kSmemLimit - 2048 - scratch) / p->slot_bytes);
  p->smem = p->nslots * p->slot_bytes + scratch;
  return 0;
}

ShapePlan shape_plan(const Plan& pl) {
  ShapePlan sp{};
  sp.G = pl.G;
  sp.NT = pl.NT;
  sp.HG = pl.HG;
  sp.NHG = pl.NHG;
  return sp;
}

cudaError_t sm_count(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
}

DeviceOnce g_smem_once;

cudaError_t set_smem_limits() {
  return g_smem_once.run([] {
    const int bytes = kSmemLimit - 2048;
    cudaError_t e = cudaFuncSetAttribute(kv4_decode_kernel<1>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kv4_decode_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               bytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kv4_decode_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               bytes);
    return e;
  });
}

}  // namespace
}  // namespace kv4
}  // namespace gqa

extern "C" {

size_t kv4_tile_bytes(int group) {
  return gqa::kv4::valid_group(group) ? static_cast<size_t>(gqa::kv4::tile_bytes(group)) : 0;
}

size_t kv4_decode_workspace_bytes(int B, int Hq, int Hkv, int group) {
  using namespace gqa::kv4;
  Plan pl;
  int sms = 0;
  if (B < 0 || make_plan(Hq, Hkv, group, &pl) != 0 || sm_count(&sms) != cudaSuccess) return 0;
  return gqa::balanced_layout(B, shape_plan(pl), gqa::balanced_grid(sms, 1)).total;
}

cudaError_t kv4_decode_launch(const gqa_bf16* q, const unsigned char* k_cache,
                              const unsigned char* v_cache, const int* block_table,
                              const int* seq_lens, gqa_bf16* out, int B, int Hq, int Hkv,
                              int group, int block_size, int max_blocks, int num_blocks,
                              float scale, void* workspace, size_t workspace_bytes,
                              cudaStream_t stream) {
  using namespace gqa::kv4;
  Plan pl;
  if (B < 0 || block_size <= 0 || block_size % kTileTokens != 0 || max_blocks <= 0 ||
      num_blocks <= 0 || make_plan(Hq, Hkv, group, &pl) != 0)
    return cudaErrorInvalidValue;
  if (B == 0) return cudaSuccess;
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out) return cudaErrorInvalidValue;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return cudaErrorMisalignedAddress;
  if (static_cast<long long>(B) * pl.NHG > INT_MAX / 2) return cudaErrorInvalidValue;
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  if ((e = set_smem_limits()) != cudaSuccess) return e;
  const int grid = gqa::balanced_grid(sms, 1);
  const gqa::BalancedLayout lay = gqa::balanced_layout(B, shape_plan(pl), grid);
  if (!workspace || workspace_bytes < lay.total || !aligned16(workspace))
    return cudaErrorInvalidValue;
  unsigned char* w = static_cast<unsigned char*>(workspace);

  DecodeParams p{};
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.out = out;
  p.part_m = reinterpret_cast<float*>(w + lay.m);
  p.part_l = reinterpret_cast<float*>(w + lay.l);
  p.part_acc = reinterpret_cast<float*>(w + lay.acc);
  p.row_info = reinterpret_cast<int2*>(w + lay.rowinfo);
  p.ends = reinterpret_cast<int2*>(w + lay.ends);
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.tiles_per_block = block_size / kTileTokens;
  p.max_blocks = max_blocks;
  p.num_blocks = num_blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.pl = pl;
  const int threads = (pl.ncw + 1) * 32;
  if (group == 32) kv4_decode_kernel<4><<<grid, threads, pl.smem, stream>>>(p);
  else if (group == 64) kv4_decode_kernel<2><<<grid, threads, pl.smem, stream>>>(p);
  else kv4_decode_kernel<1><<<grid, threads, pl.smem, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;

  gqa::CutMergeParams mp{};
  mp.row_info = p.row_info;
  mp.ends = p.ends;
  mp.part_m = p.part_m;
  mp.part_l = p.part_l;
  mp.part_acc = p.part_acc;
  mp.out = out;
  mp.rows = B * pl.NHG;
  mp.QHR = pl.HG * pl.G;
  mp.grid = grid;
  mp.out_mode = gqa::kOutBf16;
  mp.wait_ns = gqa::kWaitLimitNs;
  return gqa::launch_cut_merge(mp, sms, stream);
}

cudaError_t kv4_gather_launch(const unsigned char* k_cache, const unsigned char* v_cache,
                              const int* block_table, const int* seq_lens, const int* cu_seqlens,
                              gqa_bf16* k, gqa_bf16* v, int rows, int B, int Hkv, int group,
                              int block_size, int max_blocks, int num_blocks,
                              cudaStream_t stream) {
  using namespace gqa::kv4;
  if (rows < 0 || B < 0 || Hkv <= 0 || Hkv > 65536 || block_size <= 0 ||
      block_size % kTileTokens != 0 || max_blocks <= 0 || num_blocks <= 0 || !valid_group(group) ||
      (!cu_seqlens && rows != B))
    return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  if (!k_cache || !v_cache || !k || !v || (B > 0 && (!block_table || !seq_lens)))
    return cudaErrorInvalidValue;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k) || !aligned16(v))
    return cudaErrorMisalignedAddress;
  const gqa::Tokens tk{block_table, seq_lens, cu_seqlens, nullptr,   rows,
                       B,           max_blocks, num_blocks, block_size};
  const long long grid = (static_cast<long long>(rows) * ((Hkv + 1) / 2) + 7) / 8;
  if (grid > INT_MAX) return cudaErrorInvalidValue;
  const int g = static_cast<int>(grid);
  if (group == 32) kv4_gather_kernel<4><<<g, 256, 0, stream>>>(tk, k_cache, v_cache, k, v, Hkv);
  else if (group == 64) kv4_gather_kernel<2><<<g, 256, 0, stream>>>(tk, k_cache, v_cache, k, v, Hkv);
  else kv4_gather_kernel<1><<<g, 256, 0, stream>>>(tk, k_cache, v_cache, k, v, Hkv);
  return cudaGetLastError();
}

int kv4_decode_get_status(int reset) {
  int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess ||
      cudaMemcpyFromSymbol(&v, gqa::kv4::g_kv4_status, sizeof(int)) != cudaSuccess)
    return -1;
  if (reset) {
    const int z = 0;
    if (cudaMemcpyToSymbol(gqa::kv4::g_kv4_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // extern "C"
