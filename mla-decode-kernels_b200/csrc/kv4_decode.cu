// GQA decode over the 4-bit paged cache (include/kv4_decode.h), and the
// read-back of cached tokens as bf16.
//
// Mathematics.  Code n of K or V stands for s (n - 8) + c, s and c shared by
// the `group` dims y of a token.  With Q_y = sum of q over group y,
//     q . k_t = sum_y s_ty (sum_d q_d (n_td - 8)) + sum_y c_ty Q_y,
//     out_d   = sum_t (p_t s_ty) (n_td - 8) + sum_t p_t c_ty,
// so neither scale nor centre is ever applied to a code: K's products with
// the codes are summed per group on the tensor cores and scaled after, V's
// scales are folded into the softmax weights of each group, and both centre
// terms are one small tensor-core product per tile.
//   * K: a masked nibble is the fp16 subnormal n 2^-24 or 16 n 2^-24 as it
//     stands.  q enters in fp16, divided by a power of two per head so that
//     its largest element is in [1, 2) (and by 16 more where it meets 16 n);
//     the accumulator starts at -8 Q_y.  A q element below 2^-17 of its
//     head's largest loses bits there, 2^-25 of that largest at most.
//   * V: the nibble becomes 1024 + n or 1024 + 16 n in fp16 by one and-or,
//     then n - 8 by one packed operation, exactly.  (Codes left positive
//     would pile up a sum that the centre term takes away again: over a long
//     context fp32 loses the difference.)  The weights p_t s_ty are rounded
//     to fp16, 2^-11 instead of bf16's 2^-8.
// The softmax reference M of a head is no running maximum but any value that
// keeps the fp16 weights in range: it is set so that the largest p s is 2^9
// and moves only when one passes 2^15, so the common step takes no maximum
// and rescales nothing.
//
// Layout (one persistent CTA per SM, the balanced schedule of
// gqa_balance.cuh, cut rows merged by the cut-row merge kernel): HG x NT x TS
// = up to 16 warps: kv head, 8 of its q heads, and every TS-th pair of tiles.
// Each warp copies its own tiles (cp.async.bulk, one per tile) into its own
// ring and refills a slot as soon as it has read it, so no warp waits for
// another until the TS warps of a head meet at the end of a segment.
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
constexpr int kMaxWarps = 16;
constexpr int kMaxUnits = 4;                 // units (pairs of tiles) in a warp's ring
constexpr int kSmemLimit = 227 * 1024;
constexpr int kSmemStatic = 3 * 1024;        // bound of the kernel's static shared memory
constexpr int kPassWords = 8;                // floats per lane handed over at once at a meeting
constexpr float kNoRef = -1e30f;             // M before the first token

__device__ __forceinline__ void raise_status(int bits) { atomicOr(&g_kv4_status, bits); }

// How a launch maps to warps and shared memory (no device state).
struct Plan {
  int G, NT, HG, NHG, TS, warps;
  int units;  // ring depth
  int smem;
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

// K: codes j and j + 4 (j even), or 16 times codes j + 1 and j + 5, of a word
// shifted by 4 j, in units of 2^-24.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return w & 0x00f000f0u; }

// V: the same codes as n - 8 in fp16.  1024 + n and 1024 + 16 n are exact
// (fp16 counts in ones from 1024 on), and so is what follows.
__device__ __forceinline__ uint32_t low_centred(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64086408u));  // - 1032
  return r;
}
__device__ __forceinline__ uint32_t high_centred(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
  asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(r) : "r"(0x2c002c00u), "r"(0xd480d480u));  // / 16 - 72
  return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t max_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// D = A(16x16, row) * B(16x8, col) + D, fp16 inputs, fp32 accumulators.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
  int b, hg, row, S, s0, s1, nparts;
  long long cfirst;
};

// The CTA's share of the balanced schedule, as segments (one row, a range of
// its tiles).  Every warp keeps two in shared memory, one ahead of the other:
// for the copies and for the tiles it works on.
struct Walk {
  long long g, g_end, row0;
  int b, hg, S, L;
};

__device__ __forceinline__ int req_len(const DecodeParams& p, int b) {
  const int s = ld_nc_s32(p.seq_lens + b);
  const long long cap = static_cast<long long>(p.max_blocks) * p.tiles_per_block * kTileTokens;
  return s < 0 ? 0 : static_cast<int>(min(static_cast<long long>(s), cap));
}

__device__ __forceinline__ int tiles_of(int len) {
  return static_cast<int>((static_cast<long long>(len) + kTileTokens - 1) / kTileTokens);
}

// The next segment of the walk; row_start = its row's first tile in the
// schedule's order.  Every lane runs it on the same words.
__device__ __forceinline__ bool next_seg(Walk* wp, const DecodeParams& p, Seg& s,
                                         long long& row_start) {
  Walk w = *wp;
  bool found = false;
  while (w.g < w.g_end) {
    const long long rs = w.row0 + static_cast<long long>(w.hg) * w.L, re = rs + w.L;
    if (w.g >= re) {
      if (++w.hg == p.pl.NHG) {
        w.hg = 0;
        w.row0 += static_cast<long long>(p.pl.NHG) * w.L;
        if (++w.b >= p.B) {
          w.g = w.g_end;
          break;
        }
        w.S = req_len(p, w.b);
        w.L = tiles_of(w.S);
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
    row_start = rs;
    w.g = e;
    found = true;
    break;
  }
  __syncwarp();
  *wp = w;
  __syncwarp();
  return found;
}

__device__ __forceinline__ void group_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Units (pairs of tiles) of a segment of n tiles that warp ts of TS takes:
// units ts, ts + TS, ...
__device__ __forceinline__ int my_units(int n, int ts, int TS) {
  const int units = (n + 1) / 2;
  return ts < units ? (units - ts + TS - 1) / TS : 0;
}

// The copies of one warp: the physical tiles of its units, in order, across
// segments.  Lane i holds the tile of unit first + i / 2, i % 2 of its pair;
// the next 16 units' block ids are loaded while these are used.
struct Copier {
  const int* table;  // the segment's row of the block table
  int n, s0, hg;     // tiles of the segment, its first tile, its kv-head group
  int unit, units;   // next unit of this warp, and how many there are
  uint32_t cur, nxt; // physical tiles (block * tiles per block + place in it)

  __device__ __forceinline__ uint32_t look_up(const DecodeParams& p, int first, int ts) const {
    const int lane = threadIdx.x & 31;
    const int u = first + lane / 2;
    const int tile = 2 * (u * p.pl.TS + ts) + (lane & 1);
    if (u >= units || tile >= n) return 0;
    const int lb = (s0 + tile) / p.tiles_per_block, sub = s0 + tile - lb * p.tiles_per_block;
    int page = ld_nc_s32(table + lb);
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
      raise_status(kStatusBadPage);
      page = 0;
    }
    return static_cast<uint32_t>(page) * static_cast<uint32_t>(p.tiles_per_block) + sub;
  }

  // Tiles of the next unit (1 or 2; 0: no more), each lane's parity's tile in
  // `tile`.
  __device__ __forceinline__ int next(const DecodeParams& p, Walk* walk, int ts, uint32_t& tile) {
    while (unit == units) {
      Seg s;
      long long rs;
      if (!next_seg(walk, p, s, rs)) return 0;
      table = p.block_table + static_cast<size_t>(s.b) * p.max_blocks;
      n = s.s1 - s.s0;
      s0 = s.s0;
      hg = s.hg;
      unit = 0;
      units = my_units(n, ts, p.pl.TS);
      cur = look_up(p, 0, ts);
      nxt = look_up(p, 16, ts);
    }
    const int i = unit & 15;
    if (i == 0 && unit > 0) {
      cur = nxt;
      nxt = look_up(p, unit + 16, ts);
    }
    tile = __shfl_sync(kFull, cur, 2 * i + (threadIdx.x & 1));
    const int c = min(2, n - 2 * (unit * p.pl.TS + ts));
    ++unit;
    return c;
  }
};

// A warp's softmax state: lane (g, t) holds heads 2 t and 2 t + 1 (n = 0, 1):
// the reference M, the weights' sum l and dims 32 y + 4 g + 2 u + v in
// acc[2 y + u][2 v + n].
struct State {
  float m[2], l[2];
  float acc[8][4];
};

}  // namespace

template <int NG>
__global__ void __launch_bounds__(kMaxWarps * 32, 1)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kGroup = 128 / NG, kTile = tile_bytes(kGroup);
  constexpr uint32_t kUnit = 2 * kTile;  // K (or V) of a unit
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long sh_warp[32];
  __shared__ long long sh_info[8];
  __shared__ __align__(8) unsigned long long sh_bar[kMaxWarps][2][kMaxUnits];
  __shared__ Walk sh_walk[kMaxWarps][2];

  const Plan& pl = p.pl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int team = warp / pl.TS, ts = warp - team * pl.TS;  // team = (kv head, q-head tile)
  const int hl = team / pl.NT, j0 = (team - hl * pl.NT) * 8;
  const int cnt = min(8, pl.G - j0);
  float* const scratch = reinterpret_cast<float*>(smem + pl.warps * pl.units * 2 * kUnit) +
                         static_cast<size_t>(team) * (pl.TS / 2) * kPassWords * 32;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (lane == 0) {
    for (int i = 0; i < pl.units; ++i) {
      mbar_init(smem_u32(&sh_bar[warp][0][i]), 1);
      mbar_init(smem_u32(&sh_bar[warp][1][i]), 1);
    }
    fence_mbar_init();
  }
  balanced_start(
      p.B, pl.NHG, [&](int b) -> long long { return tiles_of(req_len(p, b)); }, sh_warp, sh_info);
  const long long E = sh_info[2], T = sh_info[5];
  if (lane < 2) {
    Walk w;
    w.g = sh_info[0];
    w.g_end = sh_info[1];
    w.b = static_cast<int>(sh_info[3]);
    w.row0 = sh_info[4] * pl.NHG;
    w.hg = 0;
    w.S = w.g < w.g_end ? req_len(p, w.b) : 0;
    w.L = tiles_of(w.S);
    sh_walk[warp][lane] = w;
  }
  __syncwarp();

  // ---- this warp's copies: unit u in slot u mod units, K and V apart ----
  const uint32_t ring = smem_u32(smem) + static_cast<uint32_t>(warp * pl.units) * 2 * kUnit;
  const uint32_t bar_k = smem_u32(&sh_bar[warp][0][0]), bar_v = smem_u32(&sh_bar[warp][1][0]);
  const uint64_t pol = policy_evict_first();
  Copier cp;
  cp.unit = cp.units = 0;
  const auto copy = [&](const unsigned char* cache, uint32_t tile, int hg, int c, uint32_t dst,
                        uint32_t bar) {
    if (lane == 0) mbar_arrive_expect_tx(bar, c * kTile);
    __syncwarp();
    if (lane < c)
      bulk_g2s(dst + lane * kTile,
               cache + (static_cast<size_t>(tile) * p.Hkv + hg * pl.HG + hl) * kTile, kTile, bar, pol);
  };
  int pending = 0;  // units copied and not yet done with
  for (int i = 0; i < pl.units; ++i) {
    uint32_t tile;
    const int c = cp.next(p, &sh_walk[warp][0], ts, tile);
    if (c == 0) break;
    copy(p.k, tile, cp.hg, c, ring + i * 2 * kUnit, bar_k + 8 * i);
    copy(p.v, tile, cp.hg, c, ring + i * 2 * kUnit + kUnit, bar_v + 8 * i);
    ++pending;
  }

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
  // After a wait gave up: waits (each with its limit) for the copies of the
  // next nk units' K and nv units' V, so that none lands after the CTA's end.
  const auto drain = [&](int nk, int nv) {
    for (int k = 0; k < max(nk, nv); ++k) {
      const bool wrap = slot + k >= pl.units;
      const int sl = wrap ? slot + k - pl.units : slot + k;
      const uint32_t ph = wrap ? phase ^ 1u : phase;
      if (k < nk) mbar_wait(bar_k + 8 * sl, ph);
      if (k < nv) mbar_wait(bar_v + 8 * sl, ph);
    }
    __syncwarp();
  };
  bool dead = false;  // a wait gave up: empty states from here on (see the K1 scan)
  bool first_seg = true;
  Seg s;
  long long row_start;
  while (next_seg(&sh_walk[warp][1], p, s, row_start)) {
    const long long row_end = row_start + tiles_of(s.S);
    s.cfirst = range_owner(row_start, T, E);
    s.nparts = static_cast<int>(range_owner(row_end - 1, T, E) - s.cfirst + 1);
    if (warp == 0 && lane == 0) {
      if (first_seg && s.nparts > 1 && row_start + s.s1 == row_end)
        p.ends[blockIdx.x] = make_int2(s.row, s.nparts);
      if (s.s0 == 0) p.row_info[s.row] = make_int2(static_cast<int>(s.cfirst), s.nparts);
    }
    first_seg = false;
    const int hbase = (s.hg * pl.HG + hl) * pl.G + j0;
    const int units = my_units(s.s1 - s.s0, ts, pl.TS);
    const int active = min(pl.TS, (s.s1 - s.s0 + 1) / 2);  // warps of the team with a unit

    State a;
    a.m[0] = a.m[1] = kNoRef;
    a.l[0] = a.l[1] = 0.f;
    #pragma unroll
    for (int mt = 0; mt < 8; ++mt) a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;

    if (units > 0) {
      // q fragments (B operand): lane (g, t) holds head g, words 4 i + t, each
      // as the dim pairs (0, 4), (1, 5), (2, 6), (3, 7) that meet the codes.
      uint32_t qf[8][2];
      uint32_t qsum_b;     // 2^-24 Q, high and low bf16 parts, as a B operand
      float start[NG][2];  // -8 2^-24 Q of heads 2 t, 2 t + 1
      float fac[2];        // what takes a sum to the score in log2 units
      {
        const bool has = g < cnt;
        const __nv_bfloat16* qrow =
            p.q + (static_cast<size_t>(s.b) * p.Hq + hbase + (has ? g : 0)) * kHeadDim;
        uint4 w[4];
        uint32_t top = 0;  // largest |q| of the head, as bits
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = has ? __ldg(reinterpret_cast<const uint4*>(qrow + 8 * (4 * i + t)))
                     : make_uint4(0, 0, 0, 0);
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          #pragma unroll
          for (int k = 0; k < 4; ++k)
            top = max(top, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
        }
        top = max(top, __shfl_xor_sync(kFull, top, 1));
        top = max(top, __shfl_xor_sync(kFull, top, 2));
        const int e = max(-100, min(100, static_cast<int>(top >> 7) - 127));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e
        const float up = p.scale_log2 * 16777216.f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        fac[0] = __shfl_sync(kFull, up, 8 * t);
        fac[1] = __shfl_sync(kFull, up, 8 * t + 4);
        float Q[NG];
        #pragma unroll
        for (int y = 0; y < NG; ++y) Q[y] = 0.f;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          float q[8];
          float sum = 0.f;
          #pragma unroll
          for (int k = 0; k < 4; ++k) {
            q[2 * k] = __uint_as_float(u[k] << 16) * down;
            q[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u) * down;
          }
          #pragma unroll
          for (int k = 0; k < 8; ++k) sum += q[k];
          qf[2 * i][0] = pack_half2(q[0], q[4]);
          qf[2 * i][1] = pack_half2(q[1] * 0.0625f, q[5] * 0.0625f);
          qf[2 * i + 1][0] = pack_half2(q[2], q[6]);
          qf[2 * i + 1][1] = pack_half2(q[3] * 0.0625f, q[7] * 0.0625f);
          sum += __shfl_xor_sync(kFull, sum, 1);
          sum += __shfl_xor_sync(kFull, sum, 2);
          Q[i * NG / 4] += sum;
        }
        float hi[NG], lo[NG];
        #pragma unroll
        for (int y = 0; y < NG; ++y) {
          Q[y] *= 1.f / 16777216.f;
          start[y][0] = -8.f * __shfl_sync(kFull, Q[y], 8 * t);
          start[y][1] = -8.f * __shfl_sync(kFull, Q[y], 8 * t + 4);
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
      float cw[4] = {0.f, 0.f, 0.f, 0.f};  // sum_t p_t c_ty: row y = g, heads 2 t, 2 t + 1

      for (int i = 0; i < units && !dead; ++i) {
        const int tile_no = s.s0 + 2 * (i * pl.TS + ts);
        const int left = s.S - tile_no * kTileTokens;  // valid tokens from here on
        const bool two = tile_no + 1 < s.s1;
        const uint32_t kb = ring + static_cast<uint32_t>(slot) * 2 * kUnit, vb = kb + kUnit;
        float x[2][4];

        // ---- scores of two tiles ----
        if (!__all_sync(kFull, mbar_wait(bar_k + 8 * slot, phase))) {
          drain(pending, pending);
          dead = true;
          break;
        }
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          // (a unit without a second tile reads what the slot held before; its
          // scores are masked like those behind the last token)
          const uint32_t tb = kb + j * kTile;
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
            for (int k = y * (4 / NG); k < (y + 1) * (4 / NG); ++k) {
              mma_f16_16816(d, low_codes(ua[k]), low_codes(ub[k]), high_codes(ua[k]),
                            high_codes(ub[k]), qf[2 * k][0], qf[2 * k][1]);
              mma_f16_16816(d, low_codes(ua[k] >> 8), low_codes(ub[k] >> 8), high_codes(ua[k] >> 8),
                            high_codes(ub[k] >> 8), qf[2 * k + 1][0], qf[2 * k + 1][1]);
            }
            sc[0] += sa[y] * d[0];
            sc[1] += sa[y] * d[1];
            sc[2] += sb[y] * d[2];
            sc[3] += sb[y] * d[3];
          }
          #pragma unroll
          for (int k = 0; k < 4; ++k) x[j][k] = sc[k] * fac[k & 1];
        }
        if (left < 2 * kTileTokens || !two) {
          const int nv = two ? left : min(left, kTileTokens);
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (j * kTileTokens + g >= nv) x[j][0] = x[j][1] = -INFINITY;
            if (j * kTileTokens + g + 8 >= nv) x[j][2] = x[j][3] = -INFINITY;
          }
        }
        __syncwarp();  // every lane has read the K slot: refill it
        uint32_t next_tile;
        const int next_c = cp.next(p, &sh_walk[warp][0], ts, next_tile);
        if (next_c) copy(p.k, next_tile, cp.hg, next_c, kb, bar_k + 8 * slot);

        // ---- weights, and the sum over V ----
        if (!__all_sync(kFull, mbar_wait(bar_v + 8 * slot, phase))) {
          drain(pending + (next_c ? 1 : 0), pending);
          dead = true;
          break;
        }
        uint32_t pw[2][2], bw[2][2][NG];  // weights (bf16), and times the scales (fp16)
        #pragma unroll 1
        for (int pass = 0;; ++pass) {
          float sm = 0.f;
          uint32_t over = 0u;  // largest fp16 weight
          float l[2] = {0.f, 0.f}, w[2][4];
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            float sa[NG], sb[NG];
            load_scales<NG>(vb + j * kTile + scale_at(0, 0, NG) + 2 * NG * g, sa);
            load_scales<NG>(vb + j * kTile + scale_at(8, 0, NG) + 2 * NG * g, sb);
            if (left < 2 * kTileTokens || !two) {
              // what lies behind the last token may be anything
              const int nv = two ? left : min(left, kTileTokens);
              #pragma unroll
              for (int y = 0; y < NG; ++y) {
                if (j * kTileTokens + g >= nv) sa[y] = 0.f;
                if (j * kTileTokens + g + 8 >= nv) sb[y] = 0.f;
              }
            }
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[j][k] = exp2_approx(x[j][k] - a.m[k & 1]);
              l[k & 1] += w[j][k];
            }
            pw[j][0] = pack_bf16x2(w[j][0], w[j][1]);
            pw[j][1] = pack_bf16x2(w[j][2], w[j][3]);
            #pragma unroll
            for (int y = 0; y < NG; ++y) {
              sm = fmaxf(sm, fmaxf(sa[y], sb[y]));
              bw[j][0][y] = pack_half2(w[j][0] * sa[y], w[j][1] * sa[y]);
              bw[j][1][y] = pack_half2(w[j][2] * sb[y], w[j][3] * sb[y]);
              over = max_half2(over, max_half2(bw[j][0][y], bw[j][1][y]));
            }
          }
          // 2^15 in either half, or a weight sum that nears fp32's range
          const bool big = (over & 0xffffu) >= 0x7800u || over >= 0x78000000u ||
                           l[0] > 1e30f || l[1] > 1e30f;
          if (pass == 1 || !__any_sync(kFull, big)) {
            a.l[0] += l[0];
            a.l[1] += l[1];
            break;
          }
          #pragma unroll
          for (int off = 4; off < 32; off <<= 1) sm = fmaxf(sm, __shfl_xor_sync(kFull, sm, off));
          const float room = __log2f(fminf(fmaxf(sm, 1e-18f), 1e30f)) - 9.f;
          #pragma unroll
          for (int n = 0; n < 2; ++n) {
            float mx = fmaxf(fmaxf(x[0][n], x[0][2 + n]), fmaxf(x[1][n], x[1][2 + n]));
            #pragma unroll
            for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, off));
            const float m = fmaxf(a.m[n], mx + room);
            const float f = exp2_approx(a.m[n] - m);
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
        for (int j = 0; j < 2; ++j) {
          if (j == 1 && !two) break;
          const uint32_t tb = vb + j * kTile;
          const uint32_t va = tb + 128 * t + 16 * (g ^ (2 * t));
          const uint4 wa = lds128(va), wb = lds128(va + 512);
          const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
          uint32_t ca = 0u, cb = 0u;
          if (g < NG) {
            ca = lds32(tb + v_centre_at(0, 0, NG) + 32 * g + 4 * t);
            cb = lds32(tb + v_centre_at(8, 0, NG) + 32 * g + 4 * t);
          }
          const int nv = left - j * kTileTokens;
          if (nv < kTileTokens) {
            if (2 * t >= nv) ca = 0u; else if (2 * t + 1 >= nv) ca &= 0xffffu;
            if (2 * t + 8 >= nv) cb = 0u; else if (2 * t + 9 >= nv) cb &= 0xffffu;
          }
          mma_bf16_16816(cw, ca, 0u, cb, 0u, movmatrix_trans(pw[j][0]), movmatrix_trans(pw[j][1]));
          #pragma unroll
          for (int y = 0; y < NG; ++y) {
            const uint32_t b0 = movmatrix_trans(bw[j][0][y]), b1 = movmatrix_trans(bw[j][1][y]);
            #pragma unroll
            for (int k = y * (4 / NG); k < (y + 1) * (4 / NG); ++k) {
              mma_f16_16816(a.acc[2 * k], low_centred(ua[k]), high_centred(ua[k]),
                            low_centred(ub[k]), high_centred(ub[k]), b0, b1);
              mma_f16_16816(a.acc[2 * k + 1], low_centred(ua[k] >> 8), high_centred(ua[k] >> 8),
                            low_centred(ub[k] >> 8), high_centred(ub[k] >> 8), b0, b1);
            }
          }
        }
        __syncwarp();  // every lane has read the V slot
        if (next_c) copy(p.v, next_tile, cp.hg, next_c, vb, bar_v + 8 * slot);
        else --pending;
        if (++slot == pl.units) {
          slot = 0;
          phase ^= 1;
        }
      }

      // ---- the warp's own sums ----
      #pragma unroll
      for (int n = 0; n < 2; ++n) {
        #pragma unroll
        for (int off = 4; off < 32; off <<= 1) a.l[n] += __shfl_xor_sync(kFull, a.l[n], off);
        #pragma unroll
        for (int y = 0; y < NG; ++y) {
          const float c = __shfl_sync(kFull, cw[n], 4 * y + t);
          #pragma unroll
          for (int k = y * (4 / NG); k < (y + 1) * (4 / NG); ++k)
            #pragma unroll
            for (int u = 0; u < 2; ++u) {
              a.acc[2 * k + u][n] += c;
              a.acc[2 * k + u][2 + n] += c;
            }
        }
      }
    }
    if (dead) {
      if (lane == 0) raise_status(kStatusWaitTimeout);
      a.m[0] = a.m[1] = -INFINITY;
      a.l[0] = a.l[1] = 0.f;
      #pragma unroll
      for (int mt = 0; mt < 8; ++mt)
        a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;
    }

    // ---- the team meets: halves hand over to halves, a few words at a time ----
    if (active > 1) {
      for (int off = pl.TS / 2; off >= 1; off >>= 1) {
        if (off >= active) continue;  // uniform over the team
        const bool gives = ts >= off && ts < 2 * off && ts < active;
        const bool takes = ts < off && ts + off < active;
        float* box = scratch + (gives ? ts - off : (takes ? ts : 0)) * kPassWords * 32 + lane;
        float fa[2], fo[2];
        #pragma unroll
        for (int pass = 0; pass < 5; ++pass) {
          if (gives) {
            if (pass == 0) {
              #pragma unroll
              for (int n = 0; n < 2; ++n) {
                box[n * 32] = a.m[n];
                box[(2 + n) * 32] = a.l[n];
              }
            } else {
              #pragma unroll
              for (int k = 0; k < kPassWords; ++k)
                box[k * 32] = a.acc[2 * (pass - 1) + k / 4][k % 4];
            }
          }
          group_barrier(1 + team, 32 * pl.TS);
          if (takes) {
            if (pass == 0) {
              #pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float mo = box[n * 32], m = fmaxf(a.m[n], mo);
                fa[n] = a.m[n] == -INFINITY ? 0.f : exp2_approx(a.m[n] - m);
                fo[n] = mo == -INFINITY ? 0.f : exp2_approx(mo - m);
                a.m[n] = m;
                a.l[n] = a.l[n] * fa[n] + box[(2 + n) * 32] * fo[n];
              }
            } else {
              #pragma unroll
              for (int k = 0; k < kPassWords; ++k) {
                float& v = a.acc[2 * (pass - 1) + k / 4][k % 4];
                v = v * fa[k & 1] + box[k * 32] * fo[k & 1];
              }
            }
          }
          group_barrier(1 + team, 32 * pl.TS);
        }
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
        // slot of the partial state: this CTA's, of the row's (K1's layout)
        const size_t idx = (static_cast<size_t>(blockIdx.x) + s.row) * (pl.HG * pl.G) + hl * pl.G +
                           j0 + head;
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
  // kv heads per row: up to 8 warps' worth, so that at least two warps share a
  // head's tokens (with up to 64 q heads per kv head); then as many warps per
  // head as 16 allow.
  p->HG = 1;
  for (int d = 1; d <= Hkv && d * p->NT <= 8; ++d)
    if (Hkv % d == 0) p->HG = d;
  p->NHG = Hkv / p->HG;
  p->TS = 1;
  while (2 * p->TS * p->HG * p->NT <= kMaxWarps) p->TS *= 2;
  p->warps = p->HG * p->NT * p->TS;
  const int unit_bytes = 4 * tile_bytes(group);  // K and V of two tiles
  const int scratch = p->HG * p->NT * (p->TS / 2) * kPassWords * 32 * 4;
  p->units = std::min(kMaxUnits, (kSmemLimit - kSmemStatic - scratch) / (p->warps * unit_bytes));
  p->smem = p->warps * p->units * unit_bytes + scratch;
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
    const int bytes = kSmemLimit - kSmemStatic;
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
  const int threads = pl.warps * 32;
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
