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
//     n meets q - q' / 16 instead, which fp16 rounds by up to 2^-11 of it.
//     The others it holds exactly except far below the head's largest: a q
//     that meets 16 n or a byte loses bits below 2^-13 of that, 2^-21 at most,
//     one that meets n below 2^-17, 2^-25 at most.  The offset 8 is taken off
//     by the centres' product, as the centre -8 s times the sum of the rounded
//     values, which is what the codes met.
//   * V: the same four values, again raw; a byte's sum is 16 out' + out, which
//     the end resolves.  The offset 8 joins the centres, through one product
//     of the weights with a constant.  The raw sums grow with the context
//     while what remains of them need not, and fp32 would lose the difference,
//     so every kFold units the centres' sum is folded into them.
// Roundings, half a step each, beside those of q above: the weights p_t s_ty
// that meet codes to fp16, 2^-11; the weights p_t that meet centres to bf16,
// 2^-8, the widest (their range is not fp16's: p_t is 2^9 over a scale); the
// sums of q that meet centres and -8 s to two bf16 parts, 2^-17; ex2.approx,
// 2^-22.  Sums are fp32, but a tensor-core product lines its terms up by the
// operands' nominal exponents, and a subnormal's is 2^-14 whatever its value:
// what lies below 2^-39 of the largest other operand (measured) is dropped from
// each term.  For 16 tokens or dims that is up to 17 times 2^-15 of one code's
// step: 2^-11 of a tile's largest p s for an output, and in a score 2^-11 of s
// times the largest of 16 q for each of its eight products.  Against 64 bits
// the output is off by 0.0018-0.0020 (relative rms), of which its own rounding
// to bf16 is 0.0017.
// A scale that is NaN or infinite spoils all dims of its request's q heads of
// that kv head (the product with -8 has zeros that meet it); V's scales count
// in full from 1e-18 to 1e30, smaller ones lose bits in fp16 and from 1e32 on
// the products overflow.
// The softmax reference M of a head is no running maximum but any value that
// keeps the fp16 weights in range: it is set so that the largest p s is 2^9
// and moves only when one passes 2^15, so the common step takes no maximum
// and rescales nothing.
//
// Layout (one persistent CTA per SM, the balanced schedule of gqa_balance.cuh,
// or one part of a row per CTA for small batches):
//   * up to 8 consumer warps, HG x NT x TS: kv head, 8 of its q heads, and
//     every TS-th unit of 4 tiles; where TS > 1 the warps of a head keep their
//     own state and meet at the end of a segment;
//   * one copy warp: a row of HG kv heads is contiguous in the cache, so one
//     cp.async.bulk brings a tile of all of them (several tiles where a row is
//     all heads and a block holds more).  A ring slot holds K or V of 4 TS
//     tiles;
//   * three planner warps: the next segment's record and its q fragments, made
//     while the consumers work on the current one.
// The consumers need more registers than 12 warps can share evenly, so the
// copy and planner warps' group gives up some of its own.  A second kernel
// merges the rows that were cut between CTAs.
//
// Measured on one B200 (32 requests of 8192 tokens, 32 / 8 heads, group 64):
// 59.5 us in a CUDA graph (64 us call by call), 5.1 TB/s of cache, against 159
// us from the bf16 cache and a floor of 47 us.  About 11 us are the two
// launches, the first copies and the merge; the stream alone, without the
// arithmetic, takes 43 us, and what remains is latency between the dependent
// steps of a unit that does not hide behind it: 2 warps per scheduler issue in
// 43 % of its cycles (integer pipe 40 %, tensor pipe 30 %, 220 instructions per
// 16-token tile and head, of which 64 unpack codes).  More than 8 q heads per
// kv head unpack every code once per 8 of them: 112, 213 and 410 us for 16, 32
// and 64 of each kv head (the bf16 cache: 312, 615 and 1209).  Group 32 (70.5
// us) spills 40 to 56 bytes at its 168 registers.  Sixteen warps of two
// tiles at once (71 us), twelve warps (59 us on one long request, but slower on
// uneven batches for its narrower rows), and score and sum warps apart (66 us)
// were slower; fp8 products are emulated for these warp-wide instructions.
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "device_once.h"
#include "gqa_balance.cuh"
#include "gqa_internal.h"
#include "gqa_ptx.cuh"
#include "kv4_decode.h"
#include "kv4_tile.cuh"
#include "kv_tokens.cuh"
#include "launch_early.cuh"

namespace gqa {
namespace kv4 {

__device__ int g_kv4_status;

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxWarps = 8;                 // consumer warps
constexpr int kUnit = 4;                     // tiles a warp works on at once
constexpr int kMaxSlots = 16;
constexpr int kWarpStart = 512;  // requests that one warp's start of the schedule takes
constexpr int kSlack = 6;        // tiles' worth of time of a segment's start and end
constexpr int kPlanners = 3;
constexpr int kThreads = (kMaxWarps + 1 + kPlanners) * 32;  // consumers, copy warp, planners
// Registers: 384 threads at 168 are launched; 256 consumer threads at 208 and
// 128 at 88 are those 64512.
constexpr int kConsumerRegs = 208, kHelperRegs = 88;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kSmemStatic = 2 * 1024;        // bound of the kernel's static shared memory
constexpr int kQWords = 20;                  // words per lane of a team's q fragments
constexpr int kPassWords = 12;               // words per lane handed over at once at a meeting
constexpr float kNoRef = -1e30f;             // M before the first token
constexpr int kFold = 8;                     // units between two folds of the V sums

__device__ __forceinline__ void raise_status(int bits) { atomicOr(&g_kv4_status, bits); }

// How a launch maps to warps and shared memory (no device state).
struct Plan {
  int G;        // q heads per kv head
  int QP, P;    // parts of P q heads each that a kv head's group is cut into (1 for G <= 64)
  int NT;       // 8-head column tiles of a part
  int HG, NHG;  // kv heads per row, rows per request (Hkv / HG * QP)
  int TS, warps;
  int pad;      // tiles that a row counts longer than it is, for its start and end
  int meet;     // the first step of a meeting: the power of two below TS
  int slot_tiles, slot_bytes, nslots;
  int q_at, box_at, smem;  // bytes: q fragments, meeting boxes, all dynamic shared memory
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
  int2* row_info;  // per row {first CTA holding a part, parts}
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

__device__ __forceinline__ uint32_t max_bf162(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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
  int cfirst, nparts;  // first CTA that holds a part of the row, and parts
};

// The CTA's share of the schedule, as segments (one row, a range of its
// tiles).  The copy warp and each planner keep their own.
//   * Balanced (u == 0): places [g, g_end) of all rows in a line, where a row
//     takes `pad` places, for what its start costs, and then its tiles.
//   * Parts (u > 0): rows cut into parts of u tiles, one part per CTA.
struct Walk {
  long long g, g_end, row0, T, E;
  int b, hg, S, L;
  int pad;
  int u, part, parts;
};

__device__ __forceinline__ int req_len(const DecodeParams& p, int b) {
  const int s = ld_plain(p.seq_lens + b);
  const long long cap = static_cast<long long>(p.max_blocks) * p.tiles_per_block * kTileTokens;
  return s < 0 ? 0 : static_cast<int>(min(static_cast<long long>(s), cap));
}

__device__ __forceinline__ int tiles_of(int len) {
  return static_cast<int>((static_cast<long long>(len) + kTileTokens - 1) / kTileTokens);
}

__device__ __forceinline__ int places_of(int tiles, int pad) { return tiles ? tiles + pad : 0; }

// The next segment of the walk.  Every lane runs it on the same words.
// kOwners: with the row's parts (the copy warp does not need them, and their
// divisions take time before the first copy).
template <bool kOwners>
__device__ __forceinline__ bool next_seg(Walk* wp, const DecodeParams& p, Seg& s) {
  Walk w = *wp;
  bool found = false;
  while (w.g < w.g_end) {
    const int places = places_of(w.L, w.pad);
    const long long rs = w.row0 + static_cast<long long>(w.hg) * places, re = rs + places;
    if (w.g >= re) {
      if (++w.hg == p.pl.NHG) {
        w.hg = 0;
        w.row0 += static_cast<long long>(p.pl.NHG) * places;
        if (++w.b >= p.B) {
          w.g = w.g_end;
          break;
        }
        w.S = req_len(p, w.b);
        w.L = tiles_of(w.S);
      }
      continue;
    }
    const long long t0 = rs + w.pad;  // the first tile's place
    const long long e = min(w.g_end, re);
    if (e <= t0) {
      w.g = e;
      continue;
    }
    s.b = w.b;
    s.hg = w.hg;
    s.row = w.b * p.pl.NHG + w.hg;
    s.S = w.S;
    if (w.u > 0) {
      s.s0 = w.part * w.u;
      s.s1 = min(w.L, s.s0 + w.u);
      s.cfirst = static_cast<int>(blockIdx.x) - w.part;
      s.nparts = w.parts;
      w.g = w.g_end;
    } else {
      s.s0 = static_cast<int>(max(w.g, t0) - t0);
      s.s1 = static_cast<int>(e - t0);
      if (kOwners) {
        s.cfirst = static_cast<int>(range_owner(t0, w.T, w.E));
        s.nparts = static_cast<int>(range_owner(re - 1, w.T, w.E)) - s.cfirst + 1;
      }
      w.g = e;
    }
    found = true;
    break;
  }
  *wp = w;
  return found;
}

// Flags of a meeting, in shared memory: set and seen by single lanes, with a
// limit on the wait.
__device__ __forceinline__ void set_flag(uint32_t* f, uint32_t v) {
  asm volatile("st.release.cta.shared.u32 [%0], %1;" ::"r"(smem_u32(f)), "r"(v) : "memory");
}
__device__ __forceinline__ bool flag_is(const uint32_t* f, uint32_t v) {
  uint32_t x;
  asm volatile("ld.acquire.cta.shared.u32 %0, [%1];" : "=r"(x) : "r"(smem_u32(f)) : "memory");
  return x == v;
}
__device__ __forceinline__ bool wait_flag(const uint32_t* f, uint32_t v) {
  if (flag_is(f, v)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (true) {
    #pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (flag_is(f, v)) return true;
    if (global_timer_ns() - t0 > kWaitLimitNs) return false;
  }
}

// What the consumers need to know of a segment.
struct Record {
  int valid;        // 0: no more segments
  int b, hg, row;
  int tiles, tokens;  // tokens: valid ones in the tiles
  int nparts;
};

__device__ __forceinline__ long long quotient(long long a, long long b) {
  // 64-bit division takes several times as long, on the way to the first copy
  if (((a | b) >> 32) == 0)
    return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// The CTA's share, by one warp alone; every lane takes a run of requests.
//
// Balanced shares may reach over several rows, and each segment costs a start
// and an end of its own, about as much as kSlack tiles of each of a head's
// warps: a row counts that much longer than it is (64 requests of 64 to 16384
// tokens 67 -> 58.5 us, 700 of 4 to 4096 163 -> 119; with 4 and 10 instead of
// 6: 61 and 59, 127 and 115).  Where cutting every row into parts of u tiles
// gives no more than one part per CTA with u at most kSlack above the balanced
// share - a few requests - that is taken instead (four requests of up to 512
// tokens: 14.0 -> 11.3 us).  For batches above kWarpStart requests the CTA has
// made the balanced start in `info` together.
__device__ __forceinline__ void start_walk(const DecodeParams& p, const long long* info,
                                           Walk& walk) {
  const int lane = threadIdx.x & 31, NHG = p.pl.NHG;
  Walk w;
  w.hg = w.u = w.part = w.parts = 0;
  w.pad = p.pl.pad;
  if (p.B > kWarpStart) {
    w.g = info[0];
    w.g_end = info[1];
    w.E = info[2];
    w.b = static_cast<int>(info[3]);
    w.row0 = info[4] * NHG;
    w.T = info[5];
  } else {
    const int n = (p.B + 31) / 32;
    const int lo = min(p.B, lane * n), hi = min(p.B, lo + n);
    // Of a request of L tiles: its places, or its parts.
    const auto weight = [&](int b, auto parts) -> long long {
      const int L = tiles_of(req_len(p, b));
      if constexpr (decltype(parts)::value) return (L + w.u - 1) / w.u;
      return places_of(L, w.pad);
    };
    long long local, x;  // of this lane's requests, and up to its last
    int rows = 0;        // its requests with tokens
    const auto scan = [&](auto parts) {
      local = 0;
      #pragma unroll 4
      for (int b = lo; b < hi; ++b) {
        const long long m = weight(b, parts);
        local += m;
        if constexpr (!decltype(parts)::value) rows += m > 0;
      }
      x = local;
      #pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long y = __shfl_up_sync(kFull, x, off);
        if (lane >= off) x += y;
      }
      return __shfl_sync(kFull, x, 31) * NHG;
    };
    const long long grid = gridDim.x, spare = grid - static_cast<long long>(p.B) * NHG;
    w.T = scan(std::false_type{});
    if (spare > 0) {
      const long long T =
          w.T - static_cast<long long>(__reduce_add_sync(kFull, rows)) * NHG * w.pad;
      const long long u = max(static_cast<long long>(kUnit), quotient(T + spare - 1, spare));
      if (u * grid <= T + kSlack * grid) w.u = static_cast<int>(u);
    }
    if (w.u > 0) {
      w.pad = 0;
      w.E = scan(std::true_type{});  // parts, at most grid
      w.g = min(static_cast<long long>(blockIdx.x), w.E);
      w.g_end = min(blockIdx.x + 1LL, w.E);
    } else {
      // (as range_parts and range_start)
      w.E = max(1LL, min(grid, w.T / 2));
      const long long c = blockIdx.x;
      w.g = c >= w.E ? w.T : quotient(c * w.T, w.E);
      w.g_end = c + 1 >= w.E ? w.T : quotient((c + 1) * w.T, w.E);
    }
    long long before = x - local;
    const bool mine = w.g < w.g_end && w.g >= before * NHG && w.g < x * NHG;
    int b = lo;
    if (mine)
      for (; b < hi; ++b) {
        const long long m = w.u > 0 ? weight(b, std::true_type{}) : weight(b, std::false_type{});
        if (w.g < (before + m) * NHG) break;
        before += m;
      }
    const unsigned who = __ballot_sync(kFull, mine);
    const int src = who ? __ffs(who) - 1 : 0;
    w.b = __shfl_sync(kFull, b, src);
    w.row0 = __shfl_sync(kFull, before, src) * NHG;
  }
  w.S = w.g < w.g_end ? req_len(p, w.b) : 0;
  w.L = tiles_of(w.S);
  if (w.u > 0 && w.g < w.g_end) {
    w.parts = (w.L + w.u - 1) / w.u;
    w.hg = static_cast<int>(w.g - w.row0) / w.parts;
    w.part = static_cast<int>(w.g - w.row0) - w.hg * w.parts;
    // one step inside the row, for next_seg
    w.row0 = 0;
    w.g = static_cast<long long>(w.hg) * w.L;
    w.g_end = w.g + 1;
  }
  walk = w;  // every lane the same
}

// A warp's softmax state: lane (g, t) holds heads 2 t and 2 t + 1 (n = 0, 1):
// the reference M, the weights' sum l and dims 32 y + 4 g + 2 u + v in
// acc[2 y + u][2 v + n].
struct State {
  float m[2], l[2];
  float acc[8][4];
};

// q fragments (B operand) of a team: lane (g, t) holds head g, words 4 i + t, each
// as the dim pairs (0, 4), (1, 5), (2, 6), (3, 7) that meet the codes; then the
// operands that meet centres and scales, 2^-24 Q and -8 2^-24 Q of the q that
// meets the codes, and for heads 2 t and 2 t + 1 the factor that takes a sum
// to the score in log2 units.
template <int NG>
__device__ __forceinline__ void prepare_q(const DecodeParams& p, int b, int hg, int team,
                                          unsigned char* q_area) {
  const Plan& pl = p.pl;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int hl = team / pl.NT, j0 = (team - hl * pl.NT) * 8;
  const int part = hg % pl.QP * pl.P;
  const bool has = j0 + g < min(pl.P, pl.G - part);
  const uint4* qrow = reinterpret_cast<const uint4*>(
      p.q + (static_cast<size_t>(b) * p.Hq + (hg / pl.QP * pl.HG + hl) * pl.G +
             (has ? part + j0 + g : 0)) * kHeadDim);
  uint32_t* dst = reinterpret_cast<uint32_t*>(q_area + team * kQWords * 128) + lane;
  uint32_t top = 0;  // largest |q| of the head, as bits
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 w = has ? ld_plain(qrow + 4 * i + t) : make_uint4(0, 0, 0, 0);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    #pragma unroll
    for (int k = 0; k < 4; ++k) top = max(top, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
  }
  top = max(top, __shfl_xor_sync(kFull, top, 1));
  top = max(top, __shfl_xor_sync(kFull, top, 2));
  const int e = max(-100, min(100, static_cast<int>(top >> 7) - 127));
  const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e
  const float up =
      p.scale_log2 * 16777216.f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
  dst[18 * 32] = __float_as_uint(__shfl_sync(kFull, up, 8 * t));
  dst[19 * 32] = __float_as_uint(__shfl_sync(kFull, up, 8 * t + 4));
  float Q[NG], R[NG];  // sums of q, and of q as rounded, which the codes meet
  #pragma unroll
  for (int y = 0; y < NG; ++y) Q[y] = R[y] = 0.f;
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 w = has ? ld_plain(qrow + 4 * i + t) : make_uint4(0, 0, 0, 0);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float q[8];
    #pragma unroll
    for (int k = 0; k < 4; ++k) {
      q[2 * k] = __uint_as_float(u[k] << 16) * down;
      q[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u) * down;
    }
    const float h = 0.0625f;
    const uint32_t f[4] = {pack_half2(q[0], q[4]), pack_half2(q[1] * h, q[5] * h),
                           pack_half2(q[2] - q[3] * h, q[6] - q[7] * h),
                           pack_half2(q[3] * h, q[7] * h)};
    float r[4];  // sums of the pairs as rounded
    #pragma unroll
    for (int k = 0; k < 4; ++k) {
      dst[(4 * i + k) * 32] = f[k];
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&f[k]));
      r[k] = x.x + x.y;
    }
    // a code of 8 everywhere is 8 b: n meets f[0], 16 n f[1], a byte f[3] and n f[2]
    float a = (q[0] + q[4] + q[1] + q[5]) + (q[2] + q[6] + q[3] + q[7]);
    float b = r[0] + 16.f * r[1] + r[2] + 17.f * r[3];
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
  dst[16 * 32] = high_low<NG>(Q, t);
  dst[17 * 32] = high_low<NG>(R, t);
}

// The planner warps: for each segment of the CTA its record, the row's entry
// for the merge, and every team's q fragments (teams are dealt to the
// planners), one segment ahead of the consumers, who prepare the first
// segment's q themselves.
template <int NG>
__device__ __forceinline__ void plan_segments(const DecodeParams& p, Walk* walk, int me,
                                              unsigned char* q_area, Record* record,
                                              uint32_t filled, uint32_t read) {
  const Plan& pl = p.pl;
  const int lane = threadIdx.x & 31;
  bool ok = true;  // the consumers still take records
  for (uint32_t n = 0;; ++n) {
    Seg s;
    const bool more = next_seg<true>(walk, p, s);
    if (ok && n > 0) ok = __all_sync(kFull, mbar_wait(read, (n - 1) & 1u));
    if (me == 0 && lane == 0) {
      Record r{};
      if (more) {
        r.valid = 1;
        r.b = s.b;
        r.hg = s.hg;
        r.row = s.row;
        r.tiles = s.s1 - s.s0;
        r.tokens = min(s.S - s.s0 * kTileTokens, r.tiles * kTileTokens);
        r.nparts = s.nparts;
        if (s.s0 == 0) p.row_info[s.row] = make_int2(s.cfirst, s.nparts);
      }
      if (ok) *record = r;
    }
    if (more && ok && n > 0) {
      for (int team = me; team < pl.HG * pl.NT; team += kPlanners)
        prepare_q<NG>(p, s.b, s.hg, team, q_area);
    }
    __syncwarp();
    if (ok && lane == 0) mbar_arrive(filled);
    if (!more) break;
  }
  if (!ok && lane == 0) raise_status(kStatusWaitTimeout);
  if (me == 0) {
    // Requests without tokens occupy no tiles: CTA (b mod grid) zeroes them.
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
      if (req_len(p, b) != 0) continue;
      for (int i = lane; i < pl.NHG; i += 32) p.row_info[b * pl.NHG + i] = make_int2(0, 0);
      uint4* o = reinterpret_cast<uint4*>(p.out + static_cast<size_t>(b) * p.Hq * kHeadDim);
      for (int i = lane; i < p.Hq * (kHeadDim / 8); i += 32) o[i] = make_uint4(0, 0, 0, 0);
    }
  }
}

}  // namespace

// kEight: HG == 8, which makes the stride between a unit's tiles a constant (3 %
// of the time at 8 kv heads and 4 q heads each).
template <int NG, bool kEight>
__global__ void __launch_bounds__(kThreads, 1)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kGroup = 128 / NG, kTile = tile_bytes(kGroup);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long sh_warp[32];
  __shared__ long long sh_info[8];
  __shared__ __align__(8) unsigned long long sh_full[kMaxSlots], sh_empty[kMaxSlots];
  __shared__ __align__(8) unsigned long long sh_seg[3];   // record filled, read; first q ready
  __shared__ Record sh_record;
  __shared__ uint32_t sh_given[kMaxWarps], sh_taken[kMaxWarps];  // meetings

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
    mbar_init(smem_u32(&sh_seg[0]), kPlanners);
    mbar_init(smem_u32(&sh_seg[1]), pl.warps);
    mbar_init(smem_u32(&sh_seg[2]), pl.HG * pl.NT);
    fence_mbar_init();
  }
  if (threadIdx.x < kMaxWarps) sh_given[threadIdx.x] = sh_taken[threadIdx.x] = 0u;
  wait_for_stream();
  if (p.B > kWarpStart)
    balanced_start(
        p.B, pl.NHG,
        [&](int b) -> long long { return places_of(tiles_of(req_len(p, b)), pl.pad); }, sh_warp,
        sh_info);
  __syncthreads();

  if (warp >= kMaxWarps) {
    // -------------------------------- copies --------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegs));
    Walk walk;  // the same in every lane
    start_walk(p, sh_info, walk);
    if (warp > kMaxWarps) {
      plan_segments<NG>(p, &walk, warp - kMaxWarps - 1, smem + pl.q_at, &sh_record,
                        smem_u32(&sh_seg[0]), smem_u32(&sh_seg[1]));
      return;
    }
    const uint32_t row_bytes = static_cast<uint32_t>(pl.HG * kTile);
    const uint64_t pol = policy_evict_first();
    int slot = 0;
    uint32_t phase = 0;
    int issued = 0;  // slots filled, counted up to nslots
    bool ok = true;
    // Lane i looks up tile first + i of a row, a batch of tiles at a time and
    // one batch (and one segment) ahead of the copies.
    const int batch = 32 / pl.slot_tiles * pl.slot_tiles;
    const bool whole = pl.HG == p.Hkv;
    const auto look_up = [&](const Seg& q, int first) -> int {
      const int tile = first + lane;
      return tile < q.s1 ? ld_plain(p.block_table + static_cast<size_t>(q.b) * p.max_blocks +
                                     tile / p.tiles_per_block)
                         : 0;
    };
    Seg s, following;
    bool more = next_seg<false>(&walk, p, s);
    int page = more ? look_up(s, s.s0) : 0;
    while (ok && more) {
      uint32_t cur = 0u;  // block * tiles per block + place in it
      int at = 0, next_page = 0;
      for (int st = s.s0; st < s.s1 && ok; st += pl.slot_tiles) {
        if (at == batch) at = 0;
        if (at == 0) {
          if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
            raise_status(kStatusBadPage);
            page = 0;
          }
          cur = static_cast<uint32_t>(page) * p.tiles_per_block + (st + lane) % p.tiles_per_block;
          page = look_up(s, st + batch);
        }
        const int nt = min(pl.slot_tiles, s.s1 - st);
        const uint32_t tile = __shfl_sync(kFull, cur, (at + lane) & 31);
        at += pl.slot_tiles;
        // A row of all kv heads goes on into the next tile of its block: one
        // copy for each run.
        int run = lane < nt ? 1 : 0;
        if (whole) {
          const int sub = (st + lane) % p.tiles_per_block;
          run = lane < nt && (lane == 0 || sub == 0) ? min(nt - lane, p.tiles_per_block - sub) : 0;
        }
        const size_t off =
            (static_cast<size_t>(tile) * p.Hkv + s.hg / pl.QP * pl.HG) * kTile;
        for (int kv = 0; kv < 2; ++kv) {
          if (!__all_sync(kFull, mbar_wait(empty + 8 * slot, phase ^ 1))) {
            raise_status(kStatusWaitTimeout);
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(full + 8 * slot, row_bytes * nt);
          __syncwarp();
          if (run > 0)
            bulk_g2s(ring + slot * pl.slot_bytes + lane * row_bytes, (kv ? p.v : p.k) + off,
                     run * row_bytes, full + 8 * slot, pol);
          issued = min(issued + 1, pl.nslots);
          if (++slot == pl.nslots) {
            slot = 0;
            phase ^= 1;
          }
        }
        if (st == s.s0) {
          more = next_seg<false>(&walk, p, following);
          next_page = more ? look_up(following, following.s0) : 0;
        }
      }
      s = following;
      page = next_page;
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
  bool dead = false;  // a wait gave up: this warp's rows are lost, and it ends
  const unsigned char* const my_q = smem + pl.q_at + team * kQWords * 128 + 4 * lane;
  uint32_t* const boxes = reinterpret_cast<uint32_t*>(smem + pl.box_at) +
                          team * (pl.TS - 1) * kPassWords * 32 + lane;  // of the team's givers
  uint32_t given = 0u;  // flag of this warp's last handing over
  for (uint32_t seg = 0; !dead; ++seg) {
    if (!__all_sync(kFull, mbar_wait(smem_u32(&sh_seg[0]), seg & 1u))) {
      dead = true;
      break;
    }
    const Record r = sh_record;
    if (!r.valid) break;
    if (seg == 0) {
      if (ts == 0) {
        prepare_q<NG>(p, r.b, r.hg, team, smem + pl.q_at);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh_seg[2]));
      }
      if (!__all_sync(kFull, mbar_wait(smem_u32(&sh_seg[2]), 0u))) {
        dead = true;
        break;
      }
    }
    uint32_t qf[8][2], qc, qs;
    float fac[2];
    #pragma unroll
    for (int i = 0; i < 16; ++i) qf[i / 2][i % 2] = lds32(my_q + 128 * i);
    qc = lds32(my_q + 128 * 16);
    qs = lds32(my_q + 128 * 17);
    fac[0] = __uint_as_float(lds32(my_q + 128 * 18));
    fac[1] = __uint_as_float(lds32(my_q + 128 * 19));
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh_seg[1]));

    State a;
    a.m[0] = a.m[1] = kNoRef;
    a.l[0] = a.l[1] = 0.f;
    #pragma unroll
    for (int mt = 0; mt < 8; ++mt) a.acc[mt][0] = a.acc[mt][1] = a.acc[mt][2] = a.acc[mt][3] = 0.f;
    // sum_t p_t (c_ty - 8 s_ty): row y = g, heads 2 t, 2 t + 1
    float cw[4] = {0.f, 0.f, 0.f, 0.f};

    const int tile_step = kEight ? 8 * kTile : pl.HG * kTile;
    const unsigned char* const tiles = smem + (kUnit * ts * pl.HG + hl) * kTile;
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
    // One unit of tiles, `left` valid tokens in it and behind it; kTail: fewer
    // than it holds.
    const auto unit = [&](auto tail, int left) {
      constexpr bool kTail = decltype(tail)::value;
      // ---- scores ----
      if (!__all_sync(kFull, mbar_wait(full + 8 * slot, phase))) return false;
      float x[kUnit][4];
      {
        const unsigned char* kb = tiles + slot * pl.slot_bytes;
        #pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          if (kTail && j * kTileTokens >= left) break;
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
      uint32_t pw[kUnit][2], bw[kUnit][2][NG];  // weights (bf16), and times the scales (fp16)
      #pragma unroll 1
      for (int pass = 0;; ++pass) {
        uint32_t top = 0u;  // largest scales (bf16 pairs)
        float l[2] = {0.f, 0.f};
        #pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          if (kTail && j * kTileTokens >= left) break;
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
          #pragma unroll
          for (int k = 0; k < (NG + 1) / 2; ++k) top = max_bf162(top, max_bf162(sa.w[k], sb.w[k]));
          l[0] += w[0] + w[2];
          l[1] += w[1] + w[3];
          pw[j][0] = pack_bf16x2(w[0], w[1]);
          pw[j][1] = pack_bf16x2(w[2], w[3]);
          #pragma unroll
          for (int y = 0; y < NG; ++y) {
            const float fa = sa[y], fb = sb[y];
            bw[j][0][y] = pack_half2(w[0] * fa, w[1] * fa);
            bw[j][1][y] = pack_half2(w[2] * fb, w[3] * fb);
          }
        }
        // No weight is above the lane's sum of them: neither that sum times the
        // largest scale may pass 2^15, nor the sum near fp32's range.
        const float most = fmaxf(l[0], l[1]);
        const float widest = fmaxf(__uint_as_float(top << 16), __uint_as_float(top & 0xffff0000u));
        const bool big = most * widest > 32768.f || most > 1e30f;
        if (pass == 1 || !__any_sync(kFull, big)) {
          a.l[0] += l[0];
          a.l[1] += l[1];
          break;
        }
        const int valid = kTail ? left : kUnit * kTileTokens;
        float sm = 0.f;  // largest scale of a token that counts
        #pragma unroll 1
        for (int i = g; i < valid; i += 8) {
          Scales<NG> sc;
          sc.load(vb + (i / kTileTokens) * tile_step + scale_at(i % kTileTokens, 0, NG));
          #pragma unroll
          for (int y = 0; y < NG; ++y)
            if (sc[y] < 1e38f) sm = fmaxf(sm, sc[y]);  // a group of infinities sets no range
        }
        #pragma unroll
        for (int off = 4; off < 32; off <<= 1) sm = fmaxf(sm, __shfl_xor_sync(kFull, sm, off));
        const float room = __log2f(fminf(fmaxf(sm, 1e-18f), 1e30f)) - 9.f;
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
          float mx = -INFINITY;
          #pragma unroll
          for (int j = 0; j < kUnit; ++j) {
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
      for (int j = 0; j < kUnit; ++j) {
        if (kTail && j * kTileTokens >= left) break;
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

    // Tokens of the segment from this warp's next unit on; the team's warps
    // take the chunks' units in turn, and all pass every chunk.
    int left = r.tokens - kUnit * ts * kTileTokens;
    int until_fold = kFold;
    for (int chunks = (r.tiles + pl.slot_tiles - 1) / pl.slot_tiles; chunks > 0 && !dead;
         --chunks, left -= pl.slot_tiles * kTileTokens) {
      if (left >= kUnit * kTileTokens) {
        dead = !unit(std::false_type{}, left);
      } else if (left > 0) {
        dead = !unit(std::true_type{}, left);
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

    if (dead) break;

    // ---- segment epilogue: the warp's own sums, in full units ----
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

    // ---- the team meets: halves hand over to halves, in three passes ----
    const int active = min(pl.TS, (r.tiles + kUnit - 1) / kUnit);  // warps of the team with tiles
    for (int off = pl.meet; off >= 1 && !dead; off >>= 1) {
      if (ts >= off && ts < 2 * off && ts < active) {  // gives
        uint32_t* box = boxes + (ts - 1) * kPassWords * 32;
        #pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
          if (!__all_sync(kFull, wait_flag(&sh_taken[warp], given))) {
            dead = true;
            break;
          }
          #pragma unroll
          for (int k = 0; k < kPassWords; ++k) {
            const int w = pass * kPassWords + k;
            const float v = w < 2 ? a.m[w] : (w < 4 ? a.l[w - 2] : a.acc[(w - 4) / 4][w % 4]);
            box[k * 32] = __float_as_uint(v);
          }
          __syncwarp();
          given = 3 * seg + pass + 1;
          if (lane == 0) set_flag(&sh_given[warp], given);
        }
      } else if (ts < off && ts + off < active) {  // takes
        const uint32_t* box = boxes + (ts + off - 1) * kPassWords * 32;
        float fa[2], fo[2];
        #pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
          if (!__all_sync(kFull, wait_flag(&sh_given[warp + off], 3 * seg + pass + 1))) {
            dead = true;
            break;
          }
          #pragma unroll
          for (int k = 0; k < kPassWords; ++k) {
            const int w = pass * kPassWords + k;
            const float v = __uint_as_float(box[k * 32]);
            if (w < 2) {
              const float m = fmaxf(a.m[w], v);
              fa[w] = exp2_approx(a.m[w] - m);
              fo[w] = exp2_approx(v - m);
              a.m[w] = m;
            } else if (w < 4) {
              a.l[w - 2] = a.l[w - 2] * fa[w - 2] + v * fo[w - 2];
            } else {
              float& o = a.acc[(w - 4) / 4][w % 4];
              o = o * fa[w & 1] + v * fo[w & 1];
            }
          }
          __syncwarp();
          if (lane == 0) set_flag(&sh_taken[warp + off], 3 * seg + pass + 1);
        }
      }
    }
    if (ts != 0 || dead) continue;
    const int part = r.hg % pl.QP * pl.P;
    const int hbase = (r.hg / pl.QP * pl.HG + hl) * pl.G + part + j0;
    const int cnt = min(8, min(pl.P, pl.G - part) - j0);
    #pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int head = 2 * t + n;
      if (head >= cnt) continue;
      if (r.nparts == 1) {
        __nv_bfloat16* o = p.out + (static_cast<size_t>(r.b) * p.Hq + hbase + head) * kHeadDim + 4 * g;
        const float inv = 1.f / a.l[n];
        #pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<uint2*>(o + 32 * y) =
              make_uint2(pack_bf16x2(a.acc[2 * y][n] * inv, a.acc[2 * y][2 + n] * inv),
                         pack_bf16x2(a.acc[2 * y + 1][n] * inv, a.acc[2 * y + 1][2 + n] * inv));
      } else {
        // this CTA's slot of the row (K1's layout)
        const size_t idx = (static_cast<size_t>(blockIdx.x) + r.row) * (pl.HG * pl.P) + hl * pl.P +
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
  if (dead && lane == 0) raise_status(kStatusWaitTimeout);
}

struct MergeParams {
  const int2* row_info;
  const float* part_m;
  const float* part_l;
  const float* part_acc;
  __nv_bfloat16* out;
  int rows, QHR;  // rows, and q heads per row (HG * P)
  int Hq, NHG, QP, HGG, G, P;  // HGG = HG * G
};

// Merge of the rows that were cut between CTAs: part k of row r is in slot
// first + k + r.  M = max m_k, out = sum 2^(m_k - M) acc_k / sum 2^(m_k - M) l_k.
// One warp per q head, lane = 4 dims, 16 parts in flight; kWide: the CTA's
// warps take an eighth of one head's parts each and meet in shared memory.
// Launched with programmatic dependent launch behind the decode, it adds 3 us
// (32 requests of 8192 tokens cut into 148 shares).
template <bool kWide>
__global__ void __launch_bounds__(256) kv4_merge_kernel(const MergeParams p) {
  constexpr int kBatch = 16;
  __shared__ float sh_m[8], sh_l[8];
  __shared__ float4 sh_a[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = kWide ? p.QHR : (p.QHR + 7) / 8;
  const long long units = static_cast<long long>(p.rows) * per;
  wait_for_stream();
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int r = static_cast<int>(u / per);
    const int j = static_cast<int>(u - static_cast<long long>(r) * per) * (kWide ? 1 : 8) +
                  (kWide ? 0 : warp);
    const int2 info = p.row_info[r];
    const int b = r / p.NHG, hg = r - b * p.NHG, part = hg % p.QP * p.P;
    // (kWide: uniform over the CTA)
    if (info.y <= 1 || j >= (p.QP == 1 ? p.QHR : min(p.P, p.G - part))) continue;
    const int k0 = kWide ? warp * info.y / 8 : 0, k1 = kWide ? (warp + 1) * info.y / 8 : info.y;
    float M = -INFINITY, L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = k0; k < k1; k += kBatch) {
      const int n = min(kBatch, k1 - k);
      const size_t first = (static_cast<size_t>(info.x) + k + r) * p.QHR + j;
      const size_t mine = first + static_cast<size_t>(min(lane, n - 1)) * p.QHR;
      const float m = lane < n ? __ldcg(p.part_m + mine) : -INFINITY;
      const float l = lane < n ? __ldcg(p.part_l + mine) : 0.f;
      float4 x[kBatch];
      #pragma unroll
      for (int k = 0; k < kBatch; ++k)
        x[k] = __ldcg(reinterpret_cast<const float4*>(
                          p.part_acc + (first + static_cast<size_t>(min(k, n - 1)) * p.QHR) * kHeadDim) +
                      lane);
      float top = fmaxf(M, m);
      #pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
      const float f = M == -INFINITY ? 0.f : exp2f(M - top);
      const float w = lane < n ? exp2f(m - top) : 0.f;
      float s = l * w;
      #pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(kFull, s, off);
      L = L * f + s;
      a.x *= f;
      a.y *= f;
      a.z *= f;
      a.w *= f;
      #pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float wk = __shfl_sync(kFull, w, k);
        if (k < n) {
          a.x += x[k].x * wk;
          a.y += x[k].y * wk;
          a.z += x[k].z * wk;
          a.w += x[k].w * wk;
        }
      }
      M = top;
    }
    if (kWide) {
      if (lane == 0) {
        sh_m[warp] = M;
        sh_l[warp] = L;
      }
      sh_a[warp][lane] = a;
      __syncthreads();
      if (warp == 0) {
        M = sh_m[0];
        #pragma unroll
        for (int k = 1; k < 8; ++k) M = fmaxf(M, sh_m[k]);
        L = 0.f;
        a = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float f = sh_m[k] == -INFINITY ? 0.f : exp2f(sh_m[k] - M);
          const float4 x = sh_a[k][lane];
          L += sh_l[k] * f;
          a.x += x.x * f;
          a.y += x.y * f;
          a.z += x.z * f;
          a.w += x.w * f;
        }
      }
      __syncthreads();
    }
    if (!kWide || warp == 0) {
      const float inv = 1.f / L;
      *reinterpret_cast<uint2*>(
          p.out + (static_cast<size_t>(b) * p.Hq + hg / p.QP * p.HGG + part + j) * kHeadDim + 4 * lane) =
          make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
    }
  }
}

// Read-back: a warp on one token, half a warp per kv head, 8 dims per lane;
// nsplit warps share a token's heads where there are few tokens.
// Bound by latency for few tokens (32: 2.4 us) and for many (16400 tokens of 8
// heads: 21 us against 14 of bytes) by its instructions, two- and four-byte
// loads with scales and centres loaded anew in every lane: issue 62 %, integer
// pipe 59 %, DRAM 1.3 TB/s.
template <int NG>
__global__ void __launch_bounds__(256)
    kv4_gather_kernel(const __grid_constant__ Tokens tk, const unsigned char* kc,
                      const unsigned char* vc, __nv_bfloat16* k, __nv_bfloat16* v, int Hkv,
                      int nsplit) {
  constexpr int kTile = tile_bytes(128 / NG), kBatch = 2;
  const int lane = threadIdx.x & 31, l = lane & 15;
  const long long w = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  wait_for_stream();
  if (w >= static_cast<long long>(tk.rows) * nsplit) return;
  const int t = static_cast<int>(w / nsplit);
  const int step = 2 * nsplit;
  const int first = 2 * static_cast<int>(w - static_cast<long long>(t) * nsplit) + (lane >> 4);
  Place pl = find_place(tk, t);
  size_t off = 0;  // of the token's tile of head 0
  int ti = 0;
  if (pl.live) {
    if (pl.pos >= static_cast<long long>(tk.max_blocks) * tk.block_size) {
      if (lane == 0) raise_status(kStatusBadPosition);
      pl.live = false;
    } else {
      const int lb = pl.pos / tk.block_size, slot = pl.pos - lb * tk.block_size;
      int page = ld_plain(tk.block_table + static_cast<size_t>(pl.b) * tk.max_blocks + lb);
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(tk.num_blocks)) {
        if (lane == 0) raise_status(kStatusBadPage);
        page = 0;
      }
      ti = slot % kTileTokens;
      off = (static_cast<size_t>(page) * (tk.block_size / kTileTokens) + slot / kTileTokens) * Hkv *
            kTile;
    }
  }
  const int y = 8 * l * NG / 128;
  const int ck = k_word(ti, l), cv = v_half(ti, 2 * l), cv2 = v_half(ti, 2 * l + 1);
  const int sc = scale_at(ti, y, NG), zk = k_centre_at(ti, y, NG), zv = v_centre_at(ti, y, NG);
  const auto ld16 = [](const unsigned char* a) -> unsigned {
    return ld_plain(reinterpret_cast<const unsigned short*>(a));
  };
  // s (n - 8) + c: n as the last bits of 2^23 + n; the product is exact.
  const auto value = [](unsigned w, int i, unsigned s, unsigned c) {
    const float n = __uint_as_float(((w >> (4 * i)) & 15u) | 0x4b000000u) - 8388616.f;
    return fmaf(n, __uint_as_float(s << 16), __uint_as_float(c << 16));
  };
  const auto pack = [&](unsigned w, unsigned s, unsigned c) {
    unsigned r[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = pack_bf16x2(value(w, 2 * i, s, c), value(w, 2 * i + 1, s, c));
    return make_uint4(r[0], r[1], r[2], r[3]);
  };
  const size_t out = static_cast<size_t>(t) * Hkv * 128 + 8 * l;
  for (int h0 = first; h0 < Hkv; h0 += kBatch * step) {
    unsigned wk[kBatch], wv[kBatch], sk[kBatch], sv[kBatch], ok[kBatch], ov[kBatch];
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * step;
      wk[i] = wv[i] = sk[i] = sv[i] = ok[i] = ov[i] = 0u;
      if (pl.live && h < Hkv) {
        const unsigned char* a = kc + off + static_cast<size_t>(h) * kTile;
        const unsigned char* b = vc + off + static_cast<size_t>(h) * kTile;
        wk[i] = ld_plain(reinterpret_cast<const unsigned*>(a + ck));
        wv[i] = ld16(b + cv) | ld16(b + cv2) << 16;
        sk[i] = ld16(a + sc);
        ok[i] = ld16(a + zk);
        sv[i] = ld16(b + sc);
        ov[i] = ld16(b + zv);
      }
    }
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * step;
      if (h >= Hkv) break;
      *reinterpret_cast<uint4*>(k + out + static_cast<size_t>(h) * 128) = pack(wk[i], sk[i], ok[i]);
      *reinterpret_cast<uint4*>(v + out + static_cast<size_t>(h) * 128) = pack(wv[i], sv[i], ov[i]);
    }
  }
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool valid_group(int group) { return group == 32 || group == 64 || group == 128; }

// 0, or -1 for dims the kernel does not take.
int make_plan(int Hq, int Hkv, int group, Plan* p) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || !valid_group(group)) return -1;
  p->G = Hq / Hkv;
  if (p->G > 128) return -1;
  const int tiles = (p->G + 7) / 8;
  p->QP = (tiles + kMaxWarps - 1) / kMaxWarps;
  p->NT = (tiles + p->QP - 1) / p->QP;
  p->P = p->QP == 1 ? p->G : 8 * p->NT;
  // kv heads per row and warps per head: the most warps, and of those the most
  // heads.  A slot's tiles have to fit the copy warp's lanes.
  int best = 0;
  for (int d = 1; d <= Hkv && d * p->NT <= kMaxWarps; ++d) {
    const int ts = std::min(kMaxWarps / (d * p->NT), 32 / kUnit);
    if (Hkv % d == 0 && d * ts >= best) {
      best = d * ts;
      p->HG = d;
      p->TS = ts;
      p->pad = kSlack * ts;
    }
  }
  p->NHG = Hkv / p->HG * p->QP;
  p->warps = p->HG * p->NT * p->TS;
  p->meet = 0;
  for (int m = 1; m < p->TS; m *= 2) p->meet = m;
  p->slot_tiles = kUnit * p->TS;
  p->slot_bytes = p->slot_tiles * p->HG * tile_bytes(group);
  const int q_bytes = p->HG * p->NT * kQWords * 128;
  const int box_bytes = p->HG * p->NT * (p->TS - 1) * kPassWords * 128;
  p->nslots = std::min(kMaxSlots, (kSmemLimit - kSmemStatic - q_bytes - box_bytes) / p->slot_bytes);
  p->q_at = p->nslots * p->slot_bytes;
  p->box_at = p->q_at + q_bytes;
  p->smem = p->box_at + box_bytes;
  return 0;
}

ShapePlan shape_plan(const Plan& pl) {
  ShapePlan sp{};
  sp.G = pl.P;
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

cudaError_t launch_merge(const MergeParams& p, int sms, cudaStream_t stream) {
  // A warp per head reads up to 16 parts at once; with fewer rows than that
  // fills, a CTA per head shares the parts of a row among its warps.
  const bool wide = p.rows < sms / 16;
  const long long units = wide ? static_cast<long long>(p.rows) * p.QHR
                               : static_cast<long long>(p.rows) * ((p.QHR + 7) / 8);
  return launch_early(wide ? kv4_merge_kernel<true> : kv4_merge_kernel<false>,
                      static_cast<int>(std::min(units, 8LL * sms)), 256, 0, stream, p);
}

DeviceOnce g_smem_once;

using DecodeKernel = void (*)(DecodeParams);

DecodeKernel decode_kernel(int group, bool eight) {
  if (group == 32) return eight ? kv4_decode_kernel<4, true> : kv4_decode_kernel<4, false>;
  if (group == 64) return eight ? kv4_decode_kernel<2, true> : kv4_decode_kernel<2, false>;
  return eight ? kv4_decode_kernel<1, true> : kv4_decode_kernel<1, false>;
}

cudaError_t set_smem_limits() {
  return g_smem_once.run([] {
    for (int group : {32, 64, 128})
      for (bool eight : {false, true}) {
        const cudaError_t e = cudaFuncSetAttribute(decode_kernel(group, eight),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kSmemLimit - kSmemStatic);
        if (e != cudaSuccess) return e;
      }
    return cudaSuccess;
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
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.tiles_per_block = block_size / kTileTokens;
  p.max_blocks = max_blocks;
  p.num_blocks = num_blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.pl = pl;
  e = gqa::launch_early(decode_kernel(group, pl.HG == 8), grid, kThreads, pl.smem, stream, p);
  if (e != cudaSuccess) return e;

  MergeParams mp{p.row_info,     p.part_m, p.part_l, p.part_acc, out,         B * pl.NHG,
                 pl.HG * pl.P, Hq,       pl.NHG,   pl.QP,      pl.HG * pl.G, pl.G,
                 pl.P};
  return launch_merge(mp, sms, stream);
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
  // One wave of warps (eight CTAs of eight on every SM) or a warp per token.
  const int nsplit = std::max(1, std::min(148 * 64 / rows, (Hkv + 1) / 2));
  const long long grid = (static_cast<long long>(rows) * nsplit + 7) / 8;
  if (grid > INT_MAX) return cudaErrorInvalidValue;
  const auto kernel = group == 32   ? kv4_gather_kernel<4>
                      : group == 64 ? kv4_gather_kernel<2>
                                    : kv4_gather_kernel<1>;
  return gqa::launch_early(kernel, static_cast<int>(grid), 256, 0, stream, tk, k_cache, v_cache, k, v,
                           Hkv, nsplit);
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
