// Appending new tokens to the paged caches: head norm, rotation and the
// page write in one pass over q, k and v (include/kv_append.h).
//
// Mathematics, per head row x[128] of a token at position p:
//     y = x * rsqrt(mean(x^2) + eps) * w                    (q and k, optional)
//     (a, b) -> (a cos - b sin, b cos + a sin)              (first rotary_dim dims)
// then q -> q_out, and k, v -> their page, in bf16 or as 4-bit codes.
//
// The pass is bound by memory: every byte of q, k and v is read once and
// written once and nothing is kept in between.  A head row is 256 bytes, so
// half a warp holds it, 8 dims per lane: in the half layout the 4 dims of a
// rotation's first half and the 4 of its second, so that a pair never leaves
// its lane; the norm's sum is four shuffles.  A warp works on one token and
// keeps its angles, multiplied by the norm's weights, in registers over all
// the heads it takes; small calls give every warp fewer heads instead, down
// to one row per half warp, so that one token's heads run side by side.
//
// Measured on one B200 (64 / 8 heads with norms): 4 prompts of 8192 tokens
// 224 us, 6.1 TB/s of a copy's 6.45; a step of 128 tokens 4.9 us, one token
// of 32 / 8 heads 2.8 us, both a launch and the chain request -> page -> row.
// Into the 4-bit cache, 16400 tokens of 32 / 8 heads take 97 us against 57 of
// bytes: 71 % of issue slots, integer pipe 53 %, DRAM at 55 %, at 44 % of the
// warps an SM holds and with spills (below).  Latent rows: 8200 tokens with 64
// heads 27 us, 5.7 TB/s.  All in CUDA graphs; a call from the host takes 7 us.
#include <cuda_bf16.h>
#include <math.h>

#include <climits>
#include <cstdint>

#include "gqa_ptx.cuh"
#include "launch_early.cuh"
#include "kv4_tile.cuh"
#include "kv_append.h"
#include "kv_tokens.cuh"

namespace gqa {
namespace append {

__device__ int g_append_status;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kBatch = 4;     // head rows a half warp loads before it works on them
constexpr int kMlaBatch = 8;  // and a quarter warp, of 128 bytes each

enum Rope : int { kNoRope = 0, kHalves = 1, kPairs = 2 };

struct Heads {
  const __nv_bfloat16* data;
  long long tok, head;
};

struct Norm {
  const void* weight;
  int fp32;
  float eps;
};

struct GqaParams {
  Tokens tk;
  Heads q, k, v;
  Norm qn, kn;
  __nv_bfloat16* q_out;
  long long qo_tok, qo_head;
  void* k_cache;
  void* v_cache;
  const float* table;  // [max_positions, rot]
  int rot, max_positions;
  int Hq, Hkv;         // Hq = 0: no q
  int zero_skipped;
  int nsplit;          // warps per token
};

__device__ __forceinline__ void raise_status(int bits) { atomicOr(&g_append_status, bits); }

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint2 ld_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void unpack8(const uint4& r, float (&x)[8]) {
  const unsigned w[4] = {r.x, r.y, r.z, r.w};
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                    pack_bf16x2(x[6], x[7]));
}

// Weights of dims d .. d + 3.
__device__ __forceinline__ void load_weight4(const Norm& n, int d, float* w) {
  if (n.fp32) {
    const float4 a =
        ld_plain(reinterpret_cast<const float4*>(static_cast<const float*>(n.weight) + d));
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  } else {
    const uint2 a =
        ld_plain(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(n.weight) + d));
    w[0] = __uint_as_float(a.x << 16); w[1] = __uint_as_float(a.x & 0xffff0000u);
    w[2] = __uint_as_float(a.y << 16); w[3] = __uint_as_float(a.y & 0xffff0000u);
  }
}

// Cosines and sines of a lane that holds 8 dims of a head: 8 angles in the
// half layout, 4 in the interleaved one.
struct Angles {
  float c[8], s[8];
};

// l = the lane's place in its head (dims 8 l ..).
template <int MODE>
__device__ __forceinline__ void load_angles(const float* row, int rot, int l, Angles& a) {
  if (MODE == kNoRope || 8 * l >= rot) return;
  const int half = rot / 2;
  if (MODE == kHalves) {
    const int j = 8 * l < half ? 8 * l : 8 * l - half;
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = ld_plain(reinterpret_cast<const float4*>(row + j) + i);
      const float4 s = ld_plain(reinterpret_cast<const float4*>(row + half + j) + i);
      const float sg = 8 * l < half ? -1.f : 1.f;
      a.c[4 * i] = c.x; a.c[4 * i + 1] = c.y; a.c[4 * i + 2] = c.z; a.c[4 * i + 3] = c.w;
      a.s[4 * i] = sg * s.x; a.s[4 * i + 1] = sg * s.y;
      a.s[4 * i + 2] = sg * s.z; a.s[4 * i + 3] = sg * s.w;
    }
  } else {
    const float4 c = ld_plain(reinterpret_cast<const float4*>(row + 4 * l));
    const float4 s = ld_plain(reinterpret_cast<const float4*>(row + half + 4 * l));
    a.c[0] = c.x; a.c[1] = c.y; a.c[2] = c.z; a.c[3] = c.w;
    a.s[0] = s.x; a.s[1] = s.y; a.s[2] = s.z; a.s[3] = s.w;
  }
}

// Rotates x (dims 8 l .. of a head).  Every lane of the warp must call it: in
// the half layout the pair's other element is rot / 16 lanes away.  Products
// and sums are rounded one by one, in the formula's order.
template <int MODE>
__device__ __forceinline__ void rotate(float (&x)[8], const Angles& a, int rot, int l) {
  if (MODE == kNoRope) return;
  const bool in = 8 * l < rot;
  if (MODE == kHalves) {
    const int step = rot / 16, lane = threadIdx.x & 31;
    const int from = !in ? lane : (8 * l < rot / 2 ? lane + step : lane - step);
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl_sync(kFull, x[i], from);
      if (in) x[i] = __fadd_rn(__fmul_rn(x[i], a.c[i]), __fmul_rn(o, a.s[i]));
    }
  } else if (in) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x[2 * i], v = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(u, a.c[i]), __fmul_rn(v, a.s[i]));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(v, a.c[i]), __fmul_rn(u, a.s[i]));
    }
  }
}

// Minimum and maximum that keep a NaN.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// a / b from an approximate 1 / b, corrected by the remainder (Markstein's
// method): a quotient that fp32 holds exactly, such as one half way between
// two codes, comes out exactly.
__device__ __forceinline__ float quotient(float a, float b, float inv) {
  const float q = __fmul_rn(a, inv);
  return __fmaf_rn(__fmaf_rn(-q, b, a), inv, q);
}

// The 4-bit codes of x (8 dims; the group's other dims in the neighbouring
// lanes), and the group's scale and centre.  Every lane must call it.
__device__ __forceinline__ unsigned quantise(const float (&x)[8], int group, unsigned short& s16,
                                             unsigned short& c16) {
  float lo = min_nan(min_nan(x[0], x[1], x[2]), min_nan(x[3], x[4], x[5]), x[6]);
  float hi = max_nan(max_nan(x[0], x[1], x[2]), max_nan(x[3], x[4], x[5]), x[6]);
  const float o = __shfl_xor_sync(kFull, min_nan(lo, x[7], x[7]), 1);
  const float u = __shfl_xor_sync(kFull, max_nan(hi, x[7], x[7]), 1);
  lo = min_nan(lo, x[7], o);
  hi = max_nan(hi, x[7], u);
  for (int off = 2; off < group / 8; off <<= 1) {
    const float a = __shfl_xor_sync(kFull, lo, off), b = __shfl_xor_sync(kFull, hi, off);
    lo = min_nan(lo, a, a);
    hi = max_nan(hi, b, b);
  }
  // Rounded up to bf16, so that 15 steps span the group (a NaN stays one).
  const float want = quotient(__fsub_rn(hi, lo), 15.f, 1.f / 15.f);
  const float s = want != want ? want
                               : __uint_as_float((__float_as_uint(want) + 0xffffu) & 0xffff0000u);
  const __nv_bfloat16 cb = __float2bfloat16(__fadd_rn(lo, __fmul_rn(8.f, s)));
  // Where 1 / s or a quotient's remainder would leave fp32's normal numbers,
  // 2^64 times everything has the same quotients.  x - c is up x - up c in one
  // rounding, for up = 1 too, so this costs nothing per value.
  const float up = s < 0x1p-100f && s > 0.f ? 0x1p64f : 1.f;
  const float step = s * up, at = -__bfloat162float(cb) * up;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
  if (s == 0.f) inv = 0.f;  // the group is one value up to the rounding of c: n = 8
  unsigned w = 0;
  #pragma unroll
  for (int i = 6; i >= 0; i -= 2) {
    const int n0 = __float2int_rn(quotient(__fmaf_rn(x[i], up, at), step, inv));
    const int n1 = __float2int_rn(quotient(__fmaf_rn(x[i + 1], up, at), step, inv));
    // clamped to [-8, 7] and put below what is there
    asm("cvt.pack.sat.s4.s32.b32 %0, %1, %2, %0;" : "+r"(w) : "r"(n1), "r"(n0));
  }
  w ^= 0x88888888u;  // + 8
  s16 = static_cast<unsigned short>(__float_as_uint(s) >> 16);
  if (s != s) s16 = 0x7fc0;
  c16 = __bfloat16_as_ushort(cb);
  return w;
}

// How the 16 lanes of a half warp hold a head's 128 dims, as four pairs
// (a_i, b_i) each that rotate together: in the half layout dims 4 l + i and
// rot / 2 + 4 l + i for the lanes l < rot / 8 and eight consecutive dims that
// do not rotate for the others; else dims 8 l + 2 i and 8 l + 2 i + 1.
template <int MODE>
struct Lay {
  int at0, at1;  // first dims of the lane's two runs of four
  bool on;       // the lane's pairs rotate

  __device__ __forceinline__ Lay(int rot, int l) {
    on = MODE != kNoRope && l < rot / 8;
    at0 = 8 * l;
    at1 = at0 + 4;
    if (MODE == kHalves && on) {
      at0 = 4 * l;
      at1 = rot / 2 + 4 * l;
    }
  }
  __device__ __forceinline__ uint4 load(const __nv_bfloat16* row) const {
    if (MODE != kHalves) return ld_stream(row + at0);
    const uint2 x = ld_stream8(row + at0), y = ld_stream8(row + at1);
    return make_uint4(x.x, x.y, y.x, y.y);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* row, const uint4& v) const {
    if (MODE != kHalves) {
      *reinterpret_cast<uint4*>(row + at0) = v;
    } else {
      *reinterpret_cast<uint2*>(row + at0) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(row + at1) = make_uint2(v.z, v.w);
    }
  }
  // Place of element i of pair member m (0: a, 1: b) in the eight loaded values.
  static __device__ __forceinline__ constexpr int at(int i, int m) {
    return MODE == kHalves ? 4 * m + i : 2 * i + m;
  }
};

// y = f (a C - b S), f (b C' + a S'): cosines and sines times the weights, f
// the norm's factor.
struct Turn {
  float ca[4], sb[4], cb[4], sa[4];
};

template <int MODE>
__device__ __forceinline__ void make_turn(const Norm& n, const float* angles, int rot, int l,
                                          const Lay<MODE>& lay, Turn& u) {
  float w[8];
  #pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (n.weight) load_weight4(n, lay.at0, w), load_weight4(n, lay.at1, w + 4);
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (lay.on) {
    c = ld_plain(reinterpret_cast<const float4*>(angles + 4 * l));
    s = ld_plain(reinterpret_cast<const float4*>(angles + rot / 2 + 4 * l));
  }
  const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float wa = w[Lay<MODE>::at(i, 0)], wb = w[Lay<MODE>::at(i, 1)];
    u.ca[i] = wa * cc[i];
    u.sb[i] = wb * ss[i];
    u.cb[i] = wb * cc[i];
    u.sa[i] = wa * ss[i];
  }
}

// Norm and rotation of the bf16 head rows first, first + step, ... < count of
// one token; every lane of the warp takes part, half 1 one row behind half 0
// (rows may differ between the halves, `iters` may not).  At dst rows are
// dst_stride apart.
template <int MODE>
__device__ __forceinline__ void turn_rows(const Lay<MODE>& lay, const __nv_bfloat16* src,
                                          long long stride, int first, int step, int iters,
                                          int count, const Norm& n,
                                          const float* angles, int rot, __nv_bfloat16* dst,
                                          long long dst_stride) {
  const int l = threadIdx.x & 15;
  uint4 raw[kBatch];
  const auto load = [&](int i0) {
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = first + (i0 + i) * step;
      raw[i] = i0 + i < iters && r < count ? lay.load(src + r * stride) : make_uint4(0, 0, 0, 0);
    }
  };
  if (iters == 0) return;
  load(0);
  Turn u;
  make_turn<MODE>(n, angles, rot, l, lay, u);
  const bool partial = MODE != kNoRope && rot < 128;
  for (int i0 = 0; i0 < iters; i0 += kBatch) {
    if (i0) load(i0);
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i >= iters) break;
      const int r = first + (i0 + i) * step;
      float x[8];
      unpack8(raw[i], x);
      if (n.weight) {
        float ss = 0.f;
        #pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
        #pragma unroll
        for (int off = 1; off < 16; off <<= 1) ss += __shfl_xor_sync(kFull, ss, off);
        const float f = rsqrtf(fmaf(ss, 1.f / 128.f, n.eps));
        #pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= f;
      }
      float y[8];
      #pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = x[Lay<MODE>::at(j, 0)], b = x[Lay<MODE>::at(j, 1)];
        if (MODE == kNoRope) {
          y[Lay<MODE>::at(j, 0)] = a * u.ca[j];
          y[Lay<MODE>::at(j, 1)] = b * u.cb[j];
        } else {
          // (an infinity that does not rotate must not meet a sine of 0)
          const float a1 = partial && !lay.on ? 0.f : a, b1 = partial && !lay.on ? 0.f : b;
          y[Lay<MODE>::at(j, 0)] = fmaf(a, u.ca[j], -(b1 * u.sb[j]));
          y[Lay<MODE>::at(j, 1)] = fmaf(b, u.cb[j], a1 * u.sa[j]);
        }
      }
      if (r < count) lay.store(dst + r * dst_stride, pack8(y));
    }
  }
}

// K (normed, rotated) or V rows of one token into its tiles of the 4-bit
// cache; 8 consecutive dims per lane.  K's fp32 operations are rounded one by
// one, in the formula's order, so that equal inputs give equal codes wherever
// they are computed.
template <int MODE, bool kValue>
__device__ __forceinline__ void quantise_rows(const __nv_bfloat16* src, long long stride,
                                              int first, int step, int iters,
                                              int count, const Norm& n,
                                              const float* angles, int rot, unsigned char* tile,
                                              int ti, int group) {
  if (iters == 0) return;
  const int l = threadIdx.x & 15, ng = 128 / group, y = 8 * l / group;
  Angles ang;
  if (!kValue) load_angles<MODE>(angles, rot, l, ang);
  float wt[8];
  if (!kValue && n.weight) {
    load_weight4(n, 8 * l, wt);
    load_weight4(n, 8 * l + 4, wt + 4);
  }
  for (int i0 = 0; i0 < iters; i0 += kBatch) {
    uint4 raw[kBatch];
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = first + (i0 + i) * step;
      raw[i] = i0 + i < iters && r < count ? ld_stream(src + r * stride + 8 * l)
                                           : make_uint4(0, 0, 0, 0);
    }
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i >= iters) break;
      const int r = first + (i0 + i) * step;
      float x[8];
      unpack8(raw[i], x);
      if (!kValue) {
        if (n.weight) {
          float ss = 0.f;
          #pragma unroll
          for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
          #pragma unroll
          for (int off = 1; off < 16; off <<= 1) ss += __shfl_xor_sync(kFull, ss, off);
          const float f = rsqrtf(ss * (1.f / 128.f) + n.eps);
          #pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = x[j] * f * wt[j];
        }
        rotate<MODE>(x, ang, rot, l);
      }
      unsigned short s16, c16;
      const unsigned codes = quantise(x, group, s16, c16);
      if (r >= count || !tile) continue;
      unsigned char* at = tile + static_cast<size_t>(r) * kv4::tile_bytes(group);
      if (kValue) {
        *reinterpret_cast<unsigned short*>(at + kv4::v_half(ti, 2 * l)) =
            static_cast<unsigned short>(codes);
        *reinterpret_cast<unsigned short*>(at + kv4::v_half(ti, 2 * l + 1)) =
            static_cast<unsigned short>(codes >> 16);
      } else {
        *reinterpret_cast<unsigned*>(at + kv4::k_word(ti, l)) = codes;
      }
      if (8 * l % group == 0) {
        *reinterpret_cast<unsigned short*>(at + kv4::scale_at(ti, y, ng)) = s16;
        *reinterpret_cast<unsigned short*>(
            at + (kValue ? kv4::v_centre_at(ti, y, ng) : kv4::k_centre_at(ti, y, ng))) = c16;
      }
    }
  }
}

// Four CTAs per SM leave 64 registers, at which the rotating kernels spill: 48
// bytes of stores and 24 of loads into the bf16 cache, 56 and 296 (half
// layout) or 8 and 20 (interleaved) into the 4-bit one.
template <int MODE, bool KV4>
__global__ void __launch_bounds__(kThreads, 4)
    kv_append_gqa_kernel(const __grid_constant__ GqaParams p, int group) {
  const int lane = threadIdx.x & 31, l = lane & 15;
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  wait_for_stream();
  if (w >= static_cast<long long>(p.tk.rows) * p.nsplit) return;
  const int t = static_cast<int>(w / p.nsplit);
  // This half warp takes every step-th of the token's rows: q heads, k, v.
  const int step = 2 * p.nsplit;
  const int mine = 2 * static_cast<int>(w - static_cast<long long>(t) * p.nsplit) + (lane >> 4);
  const auto first = [&](int before) { return ((mine - before) % step + step) % step; };
  // Steps that bring every row's turn; none where neither half has a row.
  const auto iters = [&](int from, int count) {
    return __any_sync(kFull, from < count) ? (count + step - 1) / step : 0;
  };

  const int k_first = first(p.Hq), v_first = first(p.Hq + p.Hkv);
  const __nv_bfloat16* const q = p.q.data + t * p.q.tok;
  const __nv_bfloat16* const k = p.k.data + t * p.k.tok;
  const __nv_bfloat16* const v = p.v.data + t * p.v.tok;
  const Lay<MODE> lay(p.rot, l);

  Place pl = find_place(p.tk, t);
  int bad = 0;
  if (pl.live && (pl.pos >= static_cast<long long>(p.tk.max_blocks) * p.tk.block_size ||
                  (MODE != kNoRope && (pl.rope_pos < 0 || pl.rope_pos >= p.max_positions)))) {
    bad = kStatusBadPosition;
    pl.live = false;
  }
  int page = -1, slot = 0;
  if (pl.live) {
    const int lb = pl.pos / p.tk.block_size;
    slot = pl.pos - lb * p.tk.block_size;
    page = ld_plain(p.tk.block_table + static_cast<size_t>(pl.b) * p.tk.max_blocks + lb);
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.tk.num_blocks)) {
      bad = kStatusBadPage;
      page = -1;
    }
  }
  if (bad && mine < 2 && lane == 0) raise_status(bad);
  if (!pl.live) {
    if (p.zero_skipped)
      for (int r = mine; r < p.Hq; r += step)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_tok + r * p.qo_head + 8 * l) =
            make_uint4(0, 0, 0, 0);
    return;
  }
  const float* angles = p.table + static_cast<size_t>(MODE != kNoRope ? pl.rope_pos : 0) * p.rot;
  turn_rows<MODE>(lay, q, p.q.head, mine, step, iters(mine, p.Hq), p.Hq, p.qn, angles, p.rot,
                  p.q_out + t * p.qo_tok, p.qo_head);
  const int kn = iters(k_first, p.Hkv), vn = iters(v_first, p.Hkv);
  if (KV4) {
    const size_t tile = (static_cast<size_t>(page) * (p.tk.block_size / kv4::kTileTokens) +
                         slot / kv4::kTileTokens) * p.Hkv * kv4::tile_bytes(group);
    unsigned char* const kt = page < 0 ? nullptr : static_cast<unsigned char*>(p.k_cache) + tile;
    unsigned char* const vt = page < 0 ? nullptr : static_cast<unsigned char*>(p.v_cache) + tile;
    const int ti = slot % kv4::kTileTokens;
    quantise_rows<MODE, false>(k, p.k.head, k_first, step, kn, p.Hkv, p.kn, angles, p.rot, kt,
                               ti, group);
    quantise_rows<MODE, true>(v, p.v.head, v_first, step, vn, p.Hkv, p.kn, angles, p.rot, vt,
                              ti, group);
  } else if (page >= 0) {
    const size_t row = (static_cast<size_t>(page) * p.tk.block_size + slot) * p.Hkv * 128;
    turn_rows<MODE>(lay, k, p.k.head, k_first, step, kn, p.Hkv, p.kn, angles, p.rot,
                    static_cast<__nv_bfloat16*>(p.k_cache) + row, 128);
    __nv_bfloat16* const dst = static_cast<__nv_bfloat16*>(p.v_cache) + row + 8 * l;
    for (int r = v_first; r < p.Hkv; r += kBatch * step) {
      uint4 raw[kBatch];
      #pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (r + i * step < p.Hkv) raw[i] = ld_stream(v + (r + i * step) * p.v.head + 8 * l);
      #pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (r + i * step < p.Hkv) *reinterpret_cast<uint4*>(dst + (r + i * step) * 128) = raw[i];
    }
  }
}

struct MlaParams {
  Tokens tk;
  Heads kv_c, k_pe, q_pe;
  Norm norm;
  __nv_bfloat16* q_out;
  long long qo_tok, qo_head;
  __nv_bfloat16* cache;
  const float* table;
  int max_positions;
  int h_q;  // 0: no q
  int zero_skipped;
  int nsplit;  // warps per token: one for the latent, the others for q
};

// Latent append.  Of a token's warps the first holds the 512 latent dims, 16
// per lane, and the key's 64 rotated dims; each of the others takes every
// (nsplit - 1)-th group of four q heads (8 lanes per 64-dim head).
template <int MODE>
__global__ void __launch_bounds__(kThreads)
    kv_append_mla_kernel(const __grid_constant__ MlaParams p) {
  constexpr int kRot = 64;
  const int lane = threadIdx.x & 31, l = lane & 7;
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  wait_for_stream();
  if (w >= static_cast<long long>(p.tk.rows) * p.nsplit) return;
  const int t = static_cast<int>(w / p.nsplit);
  const int split = static_cast<int>(w - static_cast<long long>(t) * p.nsplit);
  const int step = 4 * (p.nsplit - 1), first = 4 * (split - 1);

  uint4 raw[kMlaBatch];
  auto load = [&](int base) {
    #pragma unroll
    for (int i = 0; i < kMlaBatch; ++i) {
      const int h = base + i * step + (lane >> 3);
      raw[i] = h < p.h_q ? ld_stream(p.q_pe.data + t * p.q_pe.tok + h * p.q_pe.head + 8 * l)
                         : make_uint4(0, 0, 0, 0);
    }
  };
  if (split == 0) {
    raw[0] = ld_stream(p.kv_c.data + t * p.kv_c.tok + 8 * lane);
    raw[1] = ld_stream(p.kv_c.data + t * p.kv_c.tok + 256 + 8 * lane);
    raw[2] = ld_stream(p.k_pe.data + t * p.k_pe.tok + 8 * l);
  } else {
    load(first);
  }

  Place pl = find_place(p.tk, t);
  int bad = 0;
  if (pl.live && (pl.pos >= static_cast<long long>(p.tk.max_blocks) * p.tk.block_size ||
                  (MODE != kNoRope && (pl.rope_pos < 0 || pl.rope_pos >= p.max_positions)))) {
    bad = kStatusBadPosition;
    pl.live = false;
  }
  if (!pl.live) {
    if (bad && split == 0 && lane == 0) raise_status(bad);
    if (p.zero_skipped && split > 0)
      for (int h = first + (lane >> 3); h < p.h_q; h += step)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_tok + h * p.qo_head + 8 * l) =
            make_uint4(0, 0, 0, 0);
    return;
  }
  Angles ang;
  load_angles<MODE>(p.table + static_cast<size_t>(MODE != kNoRope ? pl.rope_pos : 0) * kRot, kRot, l,
                    ang);

  if (split == 0) {
    const int lb = pl.pos / p.tk.block_size;
    const int slot = pl.pos - lb * p.tk.block_size;
    const int page = ld_plain(p.tk.block_table + static_cast<size_t>(pl.b) * p.tk.max_blocks + lb);
    float k[8];
    unpack8(raw[2], k);
    rotate<MODE>(k, ang, kRot, l);
    if (p.norm.weight) {
      float a[8], b[8], wt[8];
      unpack8(raw[0], a);
      unpack8(raw[1], b);
      float ss = 0.f;
      #pragma unroll
      for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
      #pragma unroll
      for (int off = 1; off < 32; off <<= 1) ss += __shfl_xor_sync(kFull, ss, off);
      const float f = rsqrtf(ss * (1.f / 512.f) + p.norm.eps);
      load_weight4(p.norm, 8 * lane, wt);
      load_weight4(p.norm, 8 * lane + 4, wt + 4);
      #pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = a[j] * f * wt[j];
      load_weight4(p.norm, 256 + 8 * lane, wt);
      load_weight4(p.norm, 256 + 8 * lane + 4, wt + 4);
      #pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = b[j] * f * wt[j];
      raw[0] = pack8(a);
      raw[1] = pack8(b);
    }
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.tk.num_blocks)) {
      if (lane == 0) raise_status(kStatusBadPage);
      return;
    }
    __nv_bfloat16* dst =
        p.cache + (static_cast<size_t>(page) * p.tk.block_size + slot) * (512 + kRot);
    *reinterpret_cast<uint4*>(dst + 8 * lane) = raw[0];
    *reinterpret_cast<uint4*>(dst + 256 + 8 * lane) = raw[1];
    if (lane < 8) *reinterpret_cast<uint4*>(dst + 512 + 8 * l) = pack8(k);
    return;
  }
  for (int base = first; base < p.h_q; base += kMlaBatch * step) {
    if (base != first) load(base);
    #pragma unroll
    for (int i = 0; i < kMlaBatch; ++i) {
      if (base + i * step >= p.h_q) break;
      const int h = base + i * step + (lane >> 3);
      float x[8];
      unpack8(raw[i], x);
      rotate<MODE>(x, ang, kRot, l);
      if (h < p.h_q)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_tok + h * p.qo_head + 8 * l) = pack8(x);
    }
  }
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Warps that run at once on 148 SMs (four CTAs of eight on each; the latent
// append in the half layout, with 80 registers, has three): a call of fewer
// tokens spreads each token's heads over as many as fit in that one wave.
constexpr long long kFillWarps = 148 * 32;

int pick_split(int rows, int most) {
  long long n = kFillWarps / rows;
  if (n > most) n = most;
  return n < 1 ? 1 : static_cast<int>(n);
}

// Whether [a, a + bytes) and [b, b + bytes) share memory.
bool overlap(const void* a, const void* b, unsigned long long bytes) {
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return (x > y ? x - y : y - x) < bytes;
}

cudaError_t check_tokens(const kv_append_tokens* a, Tokens* t) {
  if (!a) return cudaErrorInvalidValue;
  if (a->rows < 0 || a->batch < 0 || a->max_blocks <= 0 || a->num_blocks <= 0 || a->block_size <= 0)
    return cudaErrorInvalidValue;
  if (!a->cu_seqlens && a->rows != a->batch) return cudaErrorInvalidValue;
  if (a->rows > 0 && a->batch > 0 && (!a->block_table || !a->seq_lens))
    return cudaErrorInvalidValue;
  *t = Tokens{a->block_table, a->seq_lens, a->cu_seqlens, a->positions, a->rows,
              a->batch,       a->max_blocks, a->num_blocks, a->block_size};
  return cudaSuccess;
}

cudaError_t check_heads(const kv_append_heads& a, bool heads, Heads* h) {
  if (!a.data) return cudaErrorInvalidValue;
  if (!aligned16(a.data)) return cudaErrorMisalignedAddress;
  if (a.token_stride % 8 != 0 || (heads && a.head_stride % 8 != 0))
    return cudaErrorMisalignedAddress;
  *h = Heads{a.data, a.token_stride, heads ? a.head_stride : 0};
  return cudaSuccess;
}

cudaError_t check_norm(const kv_append_norm& a, Norm* n) {
  if (a.weight && !aligned16(a.weight)) return cudaErrorMisalignedAddress;
  *n = Norm{a.weight, a.is_fp32, a.eps};
  return cudaSuccess;
}

// Rotation mode of a launch, or -1.
int rope_mode(const kv_append_rope* r, int want_dim, const float** table, int* rot, int* max_pos) {
  *table = nullptr;
  *rot = 0;
  *max_pos = 0;
  if (!r || !r->table) return kNoRope;
  if (r->rotary_dim <= 0 || r->rotary_dim > 128 || r->rotary_dim % 16 != 0 ||
      (want_dim && r->rotary_dim != want_dim) || r->max_positions <= 0 || !aligned16(r->table))
    return -1;
  *table = r->table;
  *rot = r->rotary_dim;
  *max_pos = r->max_positions;
  return r->interleaved ? kPairs : kHalves;
}

cudaError_t append_gqa(const kv_append_tokens* tokens, const kv_append_rope* rope,
                       const kv_append_heads& q, const kv_append_heads& k,
                       const kv_append_heads& v, const kv_append_norm& q_norm,
                       const kv_append_norm& k_norm, gqa_bf16* q_out, long long qo_tok,
                       long long qo_head, int zero_skipped, void* k_cache, void* v_cache, int Hq,
                       int Hkv, int group, cudaStream_t stream) {
  GqaParams p{};
  cudaError_t e = check_tokens(tokens, &p.tk);
  if (e != cudaSuccess) return e;
  if (Hkv <= 0 || (q.data && Hq <= 0) || Hq < 0 || Hq > 65536 || Hkv > 65536)
    return cudaErrorInvalidValue;
  const int mode = rope_mode(rope, 0, &p.table, &p.rot, &p.max_positions);
  if (mode < 0) return cudaErrorInvalidValue;
  if (group && p.tk.block_size % kv4::kTileTokens != 0) return cudaErrorInvalidValue;
  if (p.tk.rows == 0) return cudaSuccess;
  if ((e = check_heads(k, true, &p.k)) != cudaSuccess) return e;
  if ((e = check_heads(v, true, &p.v)) != cudaSuccess) return e;
  if ((e = check_norm(k_norm, &p.kn)) != cudaSuccess) return e;
  if (q.data) {
    if ((e = check_heads(q, true, &p.q)) != cudaSuccess) return e;
    if ((e = check_norm(q_norm, &p.qn)) != cudaSuccess) return e;
    if (!q_out) return cudaErrorInvalidValue;
    if (!aligned16(q_out) || qo_tok % 8 != 0 || qo_head % 8 != 0)
      return cudaErrorMisalignedAddress;
    p.q_out = q_out;
    p.qo_tok = qo_tok;
    p.qo_head = qo_head;
  }
  if (!k_cache || !v_cache) return cudaErrorInvalidValue;
  if (!aligned16(k_cache) || !aligned16(v_cache)) return cudaErrorMisalignedAddress;
  const unsigned long long row_bytes = group ? kv4::tile_bytes(group) / kv4::kTileTokens : 256;
  if (overlap(k_cache, v_cache, row_bytes * p.tk.num_blocks * p.tk.block_size * Hkv))
    return cudaErrorInvalidValue;
  p.Hq = q.data ? Hq : 0;
  p.Hkv = Hkv;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.zero_skipped = zero_skipped;
  p.nsplit = pick_split(p.tk.rows, (p.Hq + 2 * Hkv + 1) / 2);
  const long long warps = static_cast<long long>(p.tk.rows) * p.nsplit;
  const long long grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > INT_MAX) return cudaErrorInvalidValue;
  using Kernel = void (*)(GqaParams, int);
  const Kernel kernels[2][3] = {
      {kv_append_gqa_kernel<kNoRope, false>, kv_append_gqa_kernel<kHalves, false>,
       kv_append_gqa_kernel<kPairs, false>},
      {kv_append_gqa_kernel<kNoRope, true>, kv_append_gqa_kernel<kHalves, true>,
       kv_append_gqa_kernel<kPairs, true>}};
  return launch_early(kernels[group ? 1 : 0][mode], static_cast<int>(grid), kThreads, 0, stream, p,
                      group);
}

}  // namespace
}  // namespace append
}  // namespace gqa

extern "C" {

cudaError_t kv_append_gqa_launch(const kv_append_tokens* tokens, const kv_append_rope* rope,
                                 kv_append_heads q, kv_append_heads k, kv_append_heads v,
                                 kv_append_norm q_norm, kv_append_norm k_norm, gqa_bf16* q_out,
                                 long long q_out_token_stride, long long q_out_head_stride,
                                 int zero_skipped, gqa_bf16* k_cache, gqa_bf16* v_cache, int Hq,
                                 int Hkv, cudaStream_t stream) {
  return gqa::append::append_gqa(tokens, rope, q, k, v, q_norm, k_norm, q_out, q_out_token_stride,
                                 q_out_head_stride, zero_skipped, k_cache, v_cache, Hq, Hkv, 0,
                                 stream);
}

cudaError_t kv_append_gqa_kv4_launch(const kv_append_tokens* tokens, const kv_append_rope* rope,
                                     kv_append_heads q, kv_append_heads k, kv_append_heads v,
                                     kv_append_norm q_norm, kv_append_norm k_norm,
                                     gqa_bf16* q_out, long long q_out_token_stride,
                                     long long q_out_head_stride, int zero_skipped,
                                     unsigned char* k_cache, unsigned char* v_cache, int Hq,
                                     int Hkv, int group, cudaStream_t stream) {
  if (group != 32 && group != 64 && group != 128) return cudaErrorInvalidValue;
  return gqa::append::append_gqa(tokens, rope, q, k, v, q_norm, k_norm, q_out, q_out_token_stride,
                                 q_out_head_stride, zero_skipped, k_cache, v_cache, Hq, Hkv, group,
                                 stream);
}

cudaError_t kv_append_mla_launch(const kv_append_tokens* tokens, const kv_append_rope* rope,
                                 kv_append_heads kv_c, kv_append_heads k_pe, kv_append_norm norm,
                                 kv_append_heads q_pe, gqa_bf16* q_pe_out,
                                 long long q_out_token_stride, long long q_out_head_stride,
                                 int zero_skipped, gqa_bf16* kv_cache, int h_q,
                                 cudaStream_t stream) {
  using namespace gqa::append;
  MlaParams p{};
  cudaError_t e = check_tokens(tokens, &p.tk);
  if (e != cudaSuccess) return e;
  if (h_q < 0 || h_q > 65536 || (q_pe.data && h_q == 0)) return cudaErrorInvalidValue;
  int rot = 0;
  const int mode = rope_mode(rope, 64, &p.table, &rot, &p.max_positions);
  if (mode < 0) return cudaErrorInvalidValue;
  if (p.tk.rows == 0) return cudaSuccess;
  if ((e = check_heads(kv_c, false, &p.kv_c)) != cudaSuccess) return e;
  if ((e = check_heads(k_pe, false, &p.k_pe)) != cudaSuccess) return e;
  if ((e = check_norm(norm, &p.norm)) != cudaSuccess) return e;
  if (q_pe.data) {
    if ((e = check_heads(q_pe, true, &p.q_pe)) != cudaSuccess) return e;
    if (!q_pe_out) return cudaErrorInvalidValue;
    if (!aligned16(q_pe_out) || q_out_token_stride % 8 != 0 || q_out_head_stride % 8 != 0)
      return cudaErrorMisalignedAddress;
    p.q_out = q_pe_out;
    p.qo_tok = q_out_token_stride;
    p.qo_head = q_out_head_stride;
  }
  if (!kv_cache) return cudaErrorInvalidValue;
  if (!aligned16(kv_cache)) return cudaErrorMisalignedAddress;
  p.cache = kv_cache;
  p.h_q = q_pe.data ? h_q : 0;
  p.zero_skipped = zero_skipped;
  p.nsplit = 1 + (p.h_q ? pick_split(p.tk.rows, (p.h_q + 3) / 4) : 0);
  const long long warps = static_cast<long long>(p.tk.rows) * p.nsplit;
  const long long grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > INT_MAX) return cudaErrorInvalidValue;
  const auto kernel = mode == kNoRope   ? kv_append_mla_kernel<kNoRope>
                      : mode == kHalves ? kv_append_mla_kernel<kHalves>
                                        : kv_append_mla_kernel<kPairs>;
  return gqa::launch_early(kernel, static_cast<int>(grid), kThreads, 0, stream, p);
}

int kv_append_get_status(int reset) {
  int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess ||
      cudaMemcpyFromSymbol(&v, gqa::append::g_append_status, sizeof(int)) != cudaSuccess)
    return -1;
  if (reset) {
    const int z = 0;
    if (cudaMemcpyToSymbol(gqa::append::g_append_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // extern "C"
