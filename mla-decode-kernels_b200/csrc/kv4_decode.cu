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
//     stands, and a whole byte (16 n' + n) 2^-24.  q enters in fp16, divided
//     by a power of two per head so that its largest element is in [1, 2)
//     (and by 16 more where it meets 16 n); where n' comes with n in one byte,
//     n meets q - q' / 16 instead, which is the only one of four that fp16
//     rounds (2^-12).  A q element below 2^-17 of its head's largest loses
//     bits, 2^-25 of that largest at most.  The offset 8 is taken off by the
//     centres' product, as the centre -8 s.
//   * V: the same patterns, again raw; a byte's sum is 16 out' + out, which
//     the end resolves.  The offset 8 joins the centres, through one product
//     of the weights with a constant.  The raw sums grow with the context
//     while what remains of them need not, and fp32 would lose the difference,
//     so every kFold pairs of tiles the centres' sum is folded into them.
//     The weights p_t s_ty are rounded to fp16, 2^-11.
// The softmax reference M of a head is no running maximum but any value that
// keeps the fp16 weights in range: it is set so that the largest p s is 2^9
// and moves only when one passes 2^15, so the common step takes no maximum
// and rescales nothing.
//
// Layout (one persistent CTA per SM, the balanced schedule of
// gqa_balance.cuh, cut rows merged by the cut-row merge kernel):
//   * up to 16 consumer warps, HG x NT x TS: kv head, 8 of its q heads, and
//     every TS-th pair of tiles; the TS warps of a head keep their own state
//     and meet at the end of a segment;
//   * one copy warp: a row of HG kv heads is contiguous in the cache, so one
//     cp.async.bulk brings a tile of all of them.  A ring slot holds K or V
//     of 2 TS tiles.  The consumers need more registers than 17 warps can
//     share evenly, so the copy warp's group gives up most of its own.
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <type_traits>
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
constexpr int kMaxSlots = 16;
constexpr int kThreads = (kMaxWarps + 4) * 32;  // and the copy warp's group
// Registers: 640 threads at 96 are launched; 512 consumer threads at 112 and
// 128 at 24 are 60416 of those 61440.
constexpr int kConsumerRegs = 112, kCopyRegs = 24;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kSmemStatic = 3 * 1024;        // bound of the kernel's static shared memory
constexpr int kPassWords = 8;                // floats per lane handed over at once at a meeting
constexpr float kNoRef = -1e30f;             // M before the first token
constexpr int kFold = 16;                    // pairs of tiles between two folds of the V sums

__device__ __forceinline__ void raise_status(int bits) { atomicOr(&g_kv4_status, bits); }

// How a launch maps to warps and shared memory (no device state).
struct Plan {
  int G, NT, HG, NHG, TS, warps;
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

// Shared-memory loads (plain ones: ordered by the waits' memory clobbers,
// free to move between them).
__device__ __forceinline__ uint4 lds128(const unsigned char* a) {
  return *reinterpret_cast<const uint4*>(a);
}
__device__ __forceinline__ uint32_t lds32(const unsigned char* a) {
  return *reinterpret_cast<const uint32_t*>(a);
}
__device__ __forceinline__ uint32_t lds16(const unsigned char* a) {
  return *reinterpret_cast<const unsigned short*>(a);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes as fp16 in units of 2^-24.  Of a 32-bit word of eight codes: n of
// nibbles 0 and 4; 16 n of nibbles 1 and 5; bytes 1 and 3 (16 n' + n: nibbles
// 3 and 7, 2 and 6); and of those, n.
__device__ __forceinline__ uint32_t codes_n(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t codes_16n(uint32_t w) { return w & 0x00f000f0u; }
__device__ __forceinline__ uint32_t codes_byte(uint32_t w) { return __byte_perm(w, 0u, 0x4341); }

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

// D = A(16x16, row) * B(16x8, col) + C, fp32 sums of fp16 or bf16 products.
// Not volatile: the operands say all that orders them.
#define KV4_MMA(name, type)                                                                     \
  __device__ __forceinline__ void name(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,    \
                                       uint32_t a3, uint32_t b0, uint32_t b1) {                 \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." type "." type ".f32 "                          \
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                       \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                        \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));                                \
  }                                                                                             \
  __device__ __forceinline__ void name##_first(float (&d)[4], uint32_t a0, uint32_t a1,         \
                                               uint32_t a2, uint32_t a3, uint32_t b0,           \
                                               uint32_t b1) {                                   \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." type "." type ".f32 "                          \
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"                   \
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                        \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));                      \
  }
KV4_MMA(mma_f16, "f16")
KV4_MMA(mma_bf16, "bf16")
#undef KV4_MMA

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The NG bf16 scales (or centres) of one token, as stored: words of two.
template <int NG>
struct Scales {
  uint32_t w[(NG + 1) / 2];
  __device__ __forceinline__ void load(const unsigned char* a) {
    if constexpr (NG == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(a);
      w[0] = v.x;
      w[1] = v.y;
    } else if constexpr (NG == 2) {
      w[0] = lds32(a);
    } else {
      w[0] = lds16(a) * 0x10001u;
    }
  }
  __device__ __forceinline__ float operator[](int y) const {
    return __uint_as_float(y & 1 ? w[y / 2] & 0xffff0000u : w[y / 2] << 16);
  }
  // What lane t holds of them as an A operand whose columns are (high, low)
  // copies: 0 .. NG - 1, 0 .. NG - 1.
  __device__ __forceinline__ uint32_t operand(int t) const {
    if constexpr (NG == 4) return t & 1 ? w[1] : w[0];
    return w[0];
  }
};

// Values Q_y as the B operand that meets Scales::operand: their high bf16
// parts, then what those leave.
template <int NG>
__device__ __forceinline__ uint32_t high_low(const float (&Q)[NG], int t) {
  float hi[NG], lo[NG];
  #pragma unroll
  for (int y = 0; y < NG; ++y) {
    hi[y] = __bfloat162float(__float2bfloat16(Q[y]));
    lo[y] = Q[y] - hi[y];
  }
  if constexpr (NG == 4) {
    const uint32_t h01 = pack_bf16x2(hi[0], hi[1]), h23 = pack_bf16x2(hi[2], hi[3]);
    const uint32_t l01 = pack_bf16x2(lo[0], lo[1]), l23 = pack_bf16x2(lo[2], lo[3]);
    return t < 2 ? (t == 0 ? h01 : h23) : (t == 2 ? l01 : l23);
  } else if constexpr (NG == 2) {
    return t == 0 ? pack_bf16x2(hi[0], hi[1]) : (t == 1 ? pack_bf16x2(lo[0], lo[1]) : 0u);
  } else {
    return t == 0 ? pack_bf16x2(hi[0], lo[0]) : 0u;
  }
}

struct Seg {
  int b, hg, row, S, s0, s1;
};

// The CTA's share of the balanced schedule, as segments (one row, a range of
// its tiles).  Every warp keeps its own, in shared memory.
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

// A warp's softmax state: lane (g, t) holds heads 2 t and 2 t + 1 (n = 0, 1):
// the reference M, the weights' sum l and dims 32 y + 4 g + 2 u + v in
// acc[2 y + u][2 v + n].
struct State {
  float m[2], l[2];
  float acc[8][4];
};

}  // namespace

template <int NG>
__global__ void __launch_bounds__(kThreads, 1)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kGroup = 128 / NG, kTile = tile_bytes(kGroup);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long sh_warp[32];
  __shared__ long long sh_info[8];
  __shared__ __align__(8) unsigned long long sh_full[kMaxSlots], sh_empty[kMaxSlots];
  __shared__ Walk sh_walk[kMaxWarps + 1];

  const Plan& pl = p.pl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem);
  const uint32_t full = smem_u32(sh_full), empty = smem_u32(sh_empty);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < pl.nslots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, pl.warps);
    }
    fence_mbar_init();
  }
  balanced_start(
      p.B, pl.NHG, [&](int b) -> long long { return tiles_of(req_len(p, b)); }, sh_warp, sh_info);
  if (threadIdx.x <= kMaxWarps) {
    Walk w;
    w.g = sh_info[0];
    w.g_end = sh_info[1];
    w.b = static_cast<int>(sh_info[3]);
    w.row0 = sh_info[4] * pl.NHG;
    w.hg = 0;
    w.S = w.g < w.g_end ? req_len(p, w.b) : 0;
    w.L = tiles_of(w.S);
    sh_walk[threadIdx.x] = w;
  }
  __syncthreads();
  Seg s;
  long long row_start;

  if (warp >= kMaxWarps) {
    // -------------------------------- copies --------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCopyRegs));
    if (warp > kMaxWarps) return;
    const uint32_t row_bytes = static_cast<uint32_t>(pl.HG * kTile);
    int slot = 0;
    uint32_t phase = 0;
    int issued = 0;  // slots filled, counted up to nslots
    bool ok = true;
    while (ok && next_seg(&sh_walk[kMaxWarps], p, s, row_start)) {
      const int* table = p.block_table + static_cast<size_t>(s.b) * p.max_blocks;
      for (int st = s.s0; st < s.s1 && ok; st += pl.slot_tiles) {
        const int nt = min(pl.slot_tiles, s.s1 - st);
        size_t off = 0;
        if (lane < nt) {
          const int lb = (st + lane) / p.tiles_per_block, sub = st + lane - lb * p.tiles_per_block;
          int page = ld_nc_s32(table + lb);
          if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
            raise_status(kStatusBadPage);
            page = 0;
          }
          off = ((static_cast<size_t>(page) * p.tiles_per_block + sub) * p.Hkv +
                 static_cast<size_t>(s.hg) * pl.HG) * kTile;
        }
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
                     row_bytes, full + 8 * slot, policy_evict_first());
          issued = min(issued + 1, pl.nslots);
          if (++slot == pl.nslots) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
    }
    // No copy may land after the CTA has exited: wait (each with its limit)
    // for the last `issued` slots (see the K1 scan).
    for (int j = 0; j < issued; ++j) {
      if (--slot < 0) {
        slot = pl.nslots - 1;
        phase ^= 1;
      }
      mbar_wait(full + 8 * slot, phase);
    }
    return;
  }

  // ------------------------------ consumers -------------------------------
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  if (warp >= pl.warps) return;
  const int g = lane >> 2, t = lane & 3;
  const int team = warp / pl.TS, ts = warp - team * pl.TS;  // team = (kv head, q-head tile)
  const int hl = team / pl.NT, j0 = (team - hl * pl.NT) * 8;
  const int cnt = min(8, pl.G - j0);

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
  const auto advance = [&]() {  // this warp has read the slot
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * slot);
    if (++slot == pl.nslots) {
      slot = 0;
      phase ^= 1;
    }
  };
  bool dead = false;  // a wait gave up: empty states from here on (see the K1 scan)
  bool first_seg = true;
  while (next_seg(&sh_walk[warp], p, s, row_start)) {
    const long long E = sh_info[2], T = sh_info[5];
    const long long row_end = row_start + tiles_of(s.S);
    const int cfirst = static_cast<int>(range_owner(row_start, T, E));
    const int nparts = static_cast<int>(range_owner(row_end - 1, T, E)) - cfirst + 1;
    if (warp == 0 && lane == 0) {
      if (first_seg && nparts > 1 && row_start + s.s1 == row_end)
        p.ends[blockIdx.x] = make_int2(s.row, nparts);
      if (s.s0 == 0) p.row_info[s.row] = make_int2(cfirst, nparts);
    }
    first_seg = false;
    const int hbase = (s.hg * pl.HG + hl) * pl.G + j0;

    // q fragments (B operand): lane (g, t) holds head g, words 4 i + t, each
    // as the dim pairs (0, 4), (1, 5), (2, 6), (3, 7) that meet the codes.
    uint32_t qf[8][2];
    uint32_t qc, qs;  // 2^-24 Q, and -8 2^-24 Q of the q that meets the codes
    float fac[2];     // what takes a sum to the score in log2 units
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
        for (int k = 0; k < 4; ++k) top = max(top, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
      }
      top = max(top, __shfl_xor_sync(kFull, top, 1));
      top = max(top, __shfl_xor_sync(kFull, top, 2));
      const int e = max(-100, min(100, static_cast<int>(top >> 7) - 127));
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e
      const float up =
          p.scale_log2 * 16777216.f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      fac[0] = __shfl_sync(kFull, up, 8 * t);
      fac[1] = __shfl_sync(kFull, up, 8 * t + 4);
      float Q[NG], R[NG];  // sums of q, and of what the roundings leave of it
      #pragma unroll
      for (int y = 0; y < NG; ++y) Q[y] = R[y] = 0.f;
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        float q[8];
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
          q[2 * k] = __uint_as_float(u[k] << 16) * down;
          q[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u) * down;
        }
        const float h = 0.0625f;
        const __half d2 = __float2half_rn(q[2] - q[3] * h), d6 = __float2half_rn(q[6] - q[7] * h);
        qf[2 * i][0] = pack_half2(q[0], q[4]);
        qf[2 * i][1] = pack_half2(q[1] * h, q[5] * h);
        qf[2 * i + 1][0] = pack_half2(__half2float(d2), __half2float(d6));
        qf[2 * i + 1][1] = pack_half2(q[3] * h, q[7] * h);
        const float rest = q[0] + q[4] + q[1] + q[5] + q[3] + q[7];
        float a = rest + (q[2] + q[6]);
        float b = rest + (__half2float(d2) + q[3] * h) + (__half2float(d6) + q[7] * h);
        #pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
          a += __shfl_xor_sync(kFull, a, off);
          b += __shfl_xor_sync(kFull, b, off);
        }
        Q[i * NG / 4] += a;
        R[i * NG / 4] += b;
      }
      #pragma unroll
      for (int y = 0; y < NG; ++y) {
        Q[y] *= 1.f / 16777216.f;
        R[y] *= -8.f / 16777216.f;
      }
      qc = high_low<NG>(Q, t);
      qs = high_low<NG>(R, t);
    }

    State a;
    a.m[0] = a.m[1] = kNoRef;
    a.l[0] = a.l[1] = 0.f;
    #pragma unroll
    for (int mt = 0; mt < 8; ++mt) a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;
    // sum_t p_t (c_ty - 8 s_ty): row y = g, heads 2 t, 2 t + 1
    float cw[4] = {0.f, 0.f, 0.f, 0.f};

    const int tile_step = pl.HG * kTile;
    const unsigned char* const tiles = smem + (2 * ts * pl.HG + hl) * kTile;
    // Adds the centres' sum to the raw sums (acc, in units of 2^-24 and, for
    // the second dim of a pair, 2^-20) and starts it again.
    const auto fold = [&]() {
      #pragma unroll
      for (int n = 0; n < 2; ++n) {
        #pragma unroll
        for (int y = 0; y < NG; ++y) {
          const float c = __shfl_sync(kFull, cw[n], 4 * y + t) * (1.f / 16777216.f);
          #pragma unroll
          for (int k = y * (4 / NG); k < (y + 1) * (4 / NG); ++k) {
            a.acc[2 * k][n] += c;
            a.acc[2 * k][2 + n] += 16.f * c;
            a.acc[2 * k + 1][n] += c;
            a.acc[2 * k + 1][2 + n] += 17.f * c;
          }
        }
        cw[n] = 0.f;
      }
    };
    // One pair of tiles, `left` valid tokens in it and behind it; kTail: fewer
    // than 32.  (Without a second tile its loads read what the slot held
    // before; those scores are masked like the ones behind the last token.)
    const auto pair = [&](auto tail, int left) {
      constexpr bool kTail = decltype(tail)::value;
      // ---- scores ----
      if (!__all_sync(kFull, mbar_wait(full + 8 * slot, phase))) return false;
      float x[2][4];
      {
        const unsigned char* kb = tiles + slot * pl.slot_bytes;
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          const unsigned char* tb = kb + j * tile_step;
          const uint4 wa = lds128(tb + 64 * g + 16 * t), wb = lds128(tb + 512 + 64 * g + 16 * t);
          const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
          Scales<NG> sa, sb, ca, cb;
          sa.load(tb + scale_at(0, 0, NG) + 2 * NG * g);
          sb.load(tb + scale_at(8, 0, NG) + 2 * NG * g);
          ca.load(tb + k_centre_at(0, 0, NG) + 2 * NG * g);
          cb.load(tb + k_centre_at(8, 0, NG) + 2 * NG * g);
          mma_bf16_first(x[j], ca.operand(t), cb.operand(t), sa.operand(t), sb.operand(t), qc, qs);
          #pragma unroll
          for (int y = 0; y < NG; ++y) {
            float d[4];
            #pragma unroll
            for (int k = y * (4 / NG); k < (y + 1) * (4 / NG); ++k) {
              const uint32_t ba = codes_byte(ua[k]), bb = codes_byte(ub[k]);
              if (k == y * (4 / NG))
                mma_f16_first(d, codes_n(ua[k]), codes_n(ub[k]), codes_16n(ua[k]), codes_16n(ub[k]),
                              qf[2 * k][0], qf[2 * k][1]);
              else
                mma_f16(d, codes_n(ua[k]), codes_n(ub[k]), codes_16n(ua[k]), codes_16n(ub[k]),
                        qf[2 * k][0], qf[2 * k][1]);
              mma_f16(d, codes_n(ba), codes_n(bb), ba, bb, qf[2 * k + 1][0], qf[2 * k + 1][1]);
            }
            x[j][0] += sa[y] * d[0];
            x[j][1] += sa[y] * d[1];
            x[j][2] += sb[y] * d[2];
            x[j][3] += sb[y] * d[3];
          }
        }
      }
      advance();

      // ---- weights ----
      if (!__all_sync(kFull, mbar_wait(full + 8 * slot, phase))) return false;
      const unsigned char* vb = tiles + slot * pl.slot_bytes;
      uint32_t pw[2][2], bw[2][2][NG];  // weights (bf16), and times the scales (fp16)
      #pragma unroll 1
      for (int pass = 0;; ++pass) {
        uint32_t over = 0u;  // largest fp16 weight
        float l[2] = {0.f, 0.f};
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          const unsigned char* tb = vb + j * tile_step;
          Scales<NG> sa, sb;
          sa.load(tb + scale_at(0, 0, NG) + 2 * NG * g);
          sb.load(tb + scale_at(8, 0, NG) + 2 * NG * g);
          float w[4];
          #pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = exp2_approx(x[j][k] * fac[k & 1] - a.m[k & 1]);
          if (kTail) {
            // what lies behind the last token may be anything
            const bool oa = j * kTileTokens + g < left, ob = j * kTileTokens + g + 8 < left;
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (!oa) w[k] = 0.f;
              if (!ob) w[2 + k] = 0.f;
            }
            #pragma unroll
            for (int k = 0; k < (NG + 1) / 2; ++k) {
              if (!oa) sa.w[k] = 0u;
              if (!ob) sb.w[k] = 0u;
            }
          }
          l[0] += w[0] + w[2];
          l[1] += w[1] + w[3];
          pw[j][0] = pack_bf16x2(w[0], w[1]);
          pw[j][1] = pack_bf16x2(w[2], w[3]);
          #pragma unroll
          for (int y = 0; y < NG; ++y) {
            const float fa = sa[y], fb = sb[y];
            bw[j][0][y] = pack_half2(w[0] * fa, w[1] * fa);
            bw[j][1][y] = pack_half2(w[2] * fb, w[3] * fb);
            over = max_half2(over, max_half2(bw[j][0][y], bw[j][1][y]));
          }
        }
        // 2^15 in either half, or a weight sum that nears fp32's range
        const bool big = (over & 0xffffu) >= 0x7800u || over >= 0x78000000u || l[0] + l[1] > 1e30f;
        if (pass == 1 || !__any_sync(kFull, big)) {
          a.l[0] += l[0];
          a.l[1] += l[1];
          break;
        }
        const int valid = kTail ? left : 2 * kTileTokens;
        float sm = 0.f;  // largest scale of a token that counts
        #pragma unroll 1
        for (int i = g; i < valid; i += 8) {
          Scales<NG> sc;
          sc.load(vb + (i / kTileTokens) * tile_step + scale_at(i % kTileTokens, 0, NG));
          #pragma unroll
          for (int y = 0; y < NG; ++y) sm = fmaxf(sm, sc[y]);
        }
        #pragma unroll
        for (int off = 4; off < 32; off <<= 1) sm = fmaxf(sm, __shfl_xor_sync(kFull, sm, off));
        const float room = __log2f(fminf(fmaxf(sm, 1e-18f), 1e30f)) - 9.f;
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
          float mx = -INFINITY;
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (j * kTileTokens + g < valid) mx = fmaxf(mx, x[j][n] * fac[n]);
            if (j * kTileTokens + g + 8 < valid) mx = fmaxf(mx, x[j][2 + n] * fac[n]);
          }
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

      // ---- the sum over V ----
      #pragma unroll
      for (int j = 0; j < 2; ++j) {
        const unsigned char* tb = vb + j * tile_step;
        const unsigned char* va = tb + 128 * t + 16 * (g ^ (2 * t));
        const uint4 wa = lds128(va), wb = lds128(va + 512);
        const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
        uint32_t ca = 0u, cb = 0u;
        if (g < NG) {
          ca = lds32(tb + v_centre_at(0, 0, NG) + 32 * g + 4 * t);
          cb = lds32(tb + v_centre_at(8, 0, NG) + 32 * g + 4 * t);
        }
        if (kTail) {
          const int nv = left - j * kTileTokens;
          if (2 * t >= nv) ca = 0u; else if (2 * t + 1 >= nv) ca &= 0xffffu;
          if (2 * t + 8 >= nv) cb = 0u; else if (2 * t + 9 >= nv) cb &= 0xffffu;
        }
        mma_bf16(cw, ca, 0u, cb, 0u, transpose8x8(pw[j][0]), transpose8x8(pw[j][1]));
        #pragma unroll
        for (int y = 0; y < NG; ++y) {
          const uint32_t b0 = transpose8x8(bw[j][0][y]), b1 = transpose8x8(bw[j][1][y]);
          const uint32_t eight = g == y ? 0xc800c800u : 0u;  // row y of -8
          mma_f16(cw, eight, 0u, eight, 0u, b0, b1);
          #pragma unroll
          for (int k = y * (4 / NG); k < (y + 1) * (4 / NG); ++k) {
            const uint32_t ba = codes_byte(ua[k]), bb = codes_byte(ub[k]);
            mma_f16(a.acc[2 * k], codes_n(ua[k]), codes_16n(ua[k]), codes_n(ub[k]), codes_16n(ub[k]),
                    b0, b1);
            mma_f16(a.acc[2 * k + 1], codes_n(ba), ba, codes_n(bb), bb, b0, b1);
          }
        }
      }
      advance();
      return true;
    };

    // Tokens of the segment from this warp's next pair on; the team's warps
    // take the chunks' pairs in turn, and all pass every chunk.
    int left = min(s.S - s.s0 * kTileTokens, (s.s1 - s.s0) * kTileTokens) - 2 * ts * kTileTokens;
    int until_fold = kFold;
    for (int chunks = (s.s1 - s.s0 + pl.slot_tiles - 1) / pl.slot_tiles; chunks > 0 && !dead;
         --chunks, left -= pl.slot_tiles * kTileTokens) {
      if (left >= 2 * kTileTokens) {
        dead = !pair(std::false_type{}, left);
      } else if (left > 0) {
        dead = !pair(std::true_type{}, left);
      } else {
        for (int kv = 0; kv < 2 && !dead; ++kv) {
          dead = !__all_sync(kFull, mbar_wait(full + 8 * slot, phase));
          if (!dead) advance();
        }
      }
      if (--until_fold == 0) {
        fold();
        until_fold = kFold;
      }
    }
    fold();

    // ---- segment epilogue: the warp's own sums, in full units ----
    if (dead) {
      if (lane == 0) raise_status(kStatusWaitTimeout);
      a.m[0] = a.m[1] = -INFINITY;
      a.l[0] = a.l[1] = 0.f;
      #pragma unroll
      for (int mt = 0; mt < 8; ++mt)
        a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;
    }
    #pragma unroll
    for (int n = 0; n < 2; ++n) {
      #pragma unroll
      for (int off = 4; off < 32; off <<= 1) a.l[n] += __shfl_xor_sync(kFull, a.l[n], off);
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        float(&e)[4] = a.acc[2 * k];
        float(&o)[4] = a.acc[2 * k + 1];
        o[2 + n] = (o[2 + n] - o[n]) * 1048576.f;  // a byte's 16 out' + out
        o[n] *= 16777216.f;
        e[2 + n] *= 1048576.f;
        e[n] *= 16777216.f;
      }
    }

    // ---- the team meets: halves hand over to halves, a few words at a time ----
    const int active = min(pl.TS, (s.s1 - s.s0 + 1) / 2);  // warps of the team with tiles
    if (active > 1) {
      float* const scratch = reinterpret_cast<float*>(smem + pl.nslots * pl.slot_bytes) +
                             team * (pl.TS / 2) * kPassWords * 32;
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
      if (nparts == 1) {
        __nv_bfloat16* o = p.out + (static_cast<size_t>(s.b) * p.Hq + hbase + head) * kHeadDim + 4 * g;
        const float inv = 1.f / a.l[n];
        #pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<uint2*>(o + 32 * y) =
              make_uint2(pack_bf16x2(a.acc[2 * y][n] * inv, a.acc[2 * y][2 + n] * inv),
                         pack_bf16x2(a.acc[2 * y + 1][n] * inv, a.acc[2 * y + 1][2 + n] * inv));
      } else {
        // this CTA's slot of the row (K1's layout)
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
  p->slot_tiles = 2 * p->TS;
  p->slot_bytes = p->slot_tiles * p->HG * tile_bytes(group);
  const int scratch = p->HG * p->NT * (p->TS / 2) * kPassWords * 32 * 4;
  p->nslots = std::min(kMaxSlots, (kSmemLimit - kSmemStatic - scratch) / p->slot_bytes);
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
  const int threads = kThreads;
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
