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
// half a warp holds it, 8 dims (16 bytes) per lane: the norm's sum is four
// shuffles, a pair of the half layout is one shuffle apart (rotary_dim / 16
// lanes) and an interleaved pair sits in one lane.  A warp works on one token
// and keeps its row of the cosine / sine table in registers over all the
// heads it takes; small calls give every warp fewer heads instead, down to
// one row per half warp, so that one token's heads run side by side.
#include <cuda_bf16.h>
#include <math.h>

#include <climits>
#include <cstdint>

#include "gqa_ptx.cuh"
#include "kv4_tile.cuh"
#include "kv_append.h"
#include "kv_tokens.cuh"

namespace gqa {
namespace append {

__device__ int g_append_status;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kBatch = 4;  // head rows a half warp loads before it works on them

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
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
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

// Weights of dims d .. d + 7.
__device__ __forceinline__ void load_weight(const Norm& n, int d, float (&w)[8]) {
  if (n.fp32) {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(n.weight) + d);
    const float4 a = __ldg(f), b = __ldg(f + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    unpack8(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(n.weight) + d)),
            w);
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
      const float4 c = __ldg(reinterpret_cast<const float4*>(row + j) + i);
      const float4 s = __ldg(reinterpret_cast<const float4*>(row + half + j) + i);
      const float sg = 8 * l < half ? -1.f : 1.f;
      a.c[4 * i] = c.x; a.c[4 * i + 1] = c.y; a.c[4 * i + 2] = c.z; a.c[4 * i + 3] = c.w;
      a.s[4 * i] = sg * s.x; a.s[4 * i + 1] = sg * s.y;
      a.s[4 * i + 2] = sg * s.z; a.s[4 * i + 3] = sg * s.w;
    }
  } else {
    const float4 c = __ldg(reinterpret_cast<const float4*>(row + 4 * l));
    const float4 s = __ldg(reinterpret_cast<const float4*>(row + half + 4 * l));
    a.c[0] = c.x; a.c[1] = c.y; a.c[2] = c.z; a.c[3] = c.w;
    a.s[0] = s.x; a.s[1] = s.y; a.s[2] = s.z; a.s[3] = s.w;
  }
}

// Rotates x (dims 8 l .. of a head) where `on`.  Every lane of the warp must
// call it: in the half layout the pair's other element is rot / 16 lanes
// away.  Products and sums are rounded one by one, in the formula's order.
template <int MODE>
__device__ __forceinline__ void rotate(float (&x)[8], const Angles& a, int rot, int l, bool on) {
  if (MODE == kNoRope) return;
  const bool in = 8 * l < rot;
  if (MODE == kHalves) {
    const int step = rot / 16, lane = threadIdx.x & 31;
    const int from = !in ? lane : (8 * l < rot / 2 ? lane + step : lane - step);
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl_sync(kFull, x[i], from);
      if (on && in) x[i] = __fadd_rn(__fmul_rn(x[i], a.c[i]), __fmul_rn(o, a.s[i]));
    }
  } else if (on && in) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x[2 * i], v = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(u, a.c[i]), __fmul_rn(v, a.s[i]));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(v, a.c[i]), __fmul_rn(u, a.s[i]));
    }
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The 4-bit codes of x (8 dims; the group's other dims in the neighbouring
// lanes), and the group's scale and centre.  Every lane must call it.
__device__ __forceinline__ unsigned quantise(const float (&x)[8], int group, unsigned short& s16,
                                             unsigned short& c16) {
  float lo = x[0], hi = x[0];
  #pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
  for (int off = 1; off < group / 8; off <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(kFull, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(kFull, hi, off));
  }
  // Rounded up to bf16, so that 15 steps span the group (a NaN stays one).
  const float want = __fdiv_rn(__fsub_rn(hi, lo), 15.f);
  const float s = want != want ? want
                               : __uint_as_float((__float_as_uint(want) + 0xffffu) & 0xffff0000u);
  const __nv_bfloat16 cb = __float2bfloat16(__fadd_rn(lo, __fmul_rn(8.f, s)));
  const float c = __bfloat162float(cb);
  unsigned w = 0;
  #pragma unroll
  for (int i = 0; i < 8; ++i) {
    // s = 0: 0 / 0 or +-y / 0; the NaN converts to 0, and the group is one
    // value up to the rounding of c
    int n = s == 0.f ? 0 : __float2int_rn(__fdiv_rn(__fsub_rn(x[i], c), s));
    n = max(-8, min(7, n)) + 8;
    w |= static_cast<unsigned>(n) << (4 * i);
  }
  s16 = static_cast<unsigned short>(__float_as_uint(s) >> 16);
  if (s != s) s16 = 0x7fc0;
  c16 = __bfloat16_as_ushort(cb);
  return w;
}

template <int MODE, bool KV4>
__global__ void __launch_bounds__(kThreads)
    kv_append_gqa_kernel(const __grid_constant__ GqaParams p, int group) {
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (w >= static_cast<long long>(p.tk.rows) * p.nsplit) return;
  const int t = static_cast<int>(w / p.nsplit);
  const int split = static_cast<int>(w - static_cast<long long>(t) * p.nsplit);
  const int nrows = p.Hq + 2 * p.Hkv;
  const int step = 2 * p.nsplit;

  // One batch of this half warp's head rows: q heads, then k, then v.
  auto src = [&](int r) {
    const __nv_bfloat16* b;
    if (r < p.Hq) b = p.q.data + t * p.q.tok + r * p.q.head;
    else if (r < p.Hq + p.Hkv) b = p.k.data + t * p.k.tok + (r - p.Hq) * p.k.head;
    else b = p.v.data + t * p.v.tok + (r - p.Hq - p.Hkv) * p.v.head;
    return b + 8 * l;
  };
  uint4 raw[kBatch];
  auto load = [&](int base) {
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = base + i * step + half;
      raw[i] = r < nrows ? ld_stream(src(r)) : make_uint4(0, 0, 0, 0);
    }
  };
  load(2 * split);  // in flight while the token's place is looked up

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
    page = __ldg(p.tk.block_table + static_cast<size_t>(pl.b) * p.tk.max_blocks + lb);
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.tk.num_blocks)) {
      bad = kStatusBadPage;
      page = -1;
    }
  }
  if (bad && split == 0 && lane == 0) raise_status(bad);
  if (!pl.live) {
    if (p.zero_skipped)
      for (int r = 2 * split + half; r < p.Hq; r += step)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_tok + r * p.qo_head + 8 * l) =
            make_uint4(0, 0, 0, 0);
    return;
  }
  Angles ang;
  load_angles<MODE>(p.table + static_cast<size_t>(MODE != kNoRope ? pl.rope_pos : 0) * p.rot, p.rot,
                    l, ang);

  for (int base = 2 * split; base < nrows; base += kBatch * step) {
    if (base != 2 * split) load(base);
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r0 = base + i * step;  // warp-uniform: the first half's row
      if (r0 >= nrows) break;
      const int r = r0 + half;
      const int kind = r < p.Hq ? 0 : (r < p.Hq + p.Hkv ? 1 : 2);
      const int h = kind == 0 ? r : (kind == 1 ? r - p.Hq : r - p.Hq - p.Hkv);
      float x[8];
      unpack8(raw[i], x);
      if (p.qn.weight || p.kn.weight) {
        float ss = 0.f;
        #pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
        #pragma unroll
        for (int off = 1; off < 16; off <<= 1) ss += __shfl_xor_sync(kFull, ss, off);
        const Norm& n = kind == 0 ? p.qn : p.kn;
        if (kind < 2 && n.weight) {
          const float f = rsqrtf(ss * (1.f / 128.f) + n.eps);
          float wt[8];
          load_weight(n, 8 * l, wt);
          #pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = x[j] * f * wt[j];
        }
      }
      rotate<MODE>(x, ang, p.rot, l, kind < 2);
      if (r < nrows && kind == 0)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_tok + h * p.qo_head + 8 * l) = pack8(x);
      if (!KV4) {
        if (r < nrows && kind > 0 && page >= 0) {
          __nv_bfloat16* c = static_cast<__nv_bfloat16*>(kind == 1 ? p.k_cache : p.v_cache);
          *reinterpret_cast<uint4*>(
              c + ((static_cast<size_t>(page) * p.tk.block_size + slot) * p.Hkv + h) * 128 + 8 * l) =
              kind == 1 ? pack8(x) : raw[i];
        }
      } else if (r0 + 1 >= p.Hq) {  // warp-uniform: one of the two rows is K or V
        unsigned short s16, c16;
        const unsigned codes = quantise(x, group, s16, c16);
        if (r < nrows && kind > 0 && page >= 0) {
          const int ng = 128 / group, y = 8 * l / group, ti = slot % kv4::kTileTokens;
          unsigned char* tile =
              static_cast<unsigned char*>(kind == 1 ? p.k_cache : p.v_cache) +
              ((static_cast<size_t>(page) * (p.tk.block_size / kv4::kTileTokens) +
                slot / kv4::kTileTokens) * p.Hkv + h) * kv4::tile_bytes(group);
          if (kind == 1) {
            *reinterpret_cast<unsigned*>(tile + kv4::k_word(ti, l)) = codes;
          } else {
            *reinterpret_cast<unsigned short*>(tile + kv4::v_half(ti, 2 * l)) =
                static_cast<unsigned short>(codes);
            *reinterpret_cast<unsigned short*>(tile + kv4::v_half(ti, 2 * l + 1)) =
                static_cast<unsigned short>(codes >> 16);
          }
          if (8 * l % group == 0) {
            *reinterpret_cast<unsigned short*>(tile + kv4::scale_at(ti, y, ng)) = s16;
            *reinterpret_cast<unsigned short*>(
                tile + (kind == 1 ? kv4::k_centre_at(ti, y, ng) : kv4::v_centre_at(ti, y, ng))) =
                c16;
          }
        }
      }
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
  if (w >= static_cast<long long>(p.tk.rows) * p.nsplit) return;
  const int t = static_cast<int>(w / p.nsplit);
  const int split = static_cast<int>(w - static_cast<long long>(t) * p.nsplit);
  const int step = 4 * (p.nsplit - 1), first = 4 * (split - 1);

  uint4 raw[kBatch];
  auto load = [&](int base) {
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
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
    const int page = __ldg(p.tk.block_table + static_cast<size_t>(pl.b) * p.tk.max_blocks + lb);
    float k[8];
    unpack8(raw[2], k);
    rotate<MODE>(k, ang, kRot, l, true);
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
      load_weight(p.norm, 8 * lane, wt);
      #pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = a[j] * f * wt[j];
      load_weight(p.norm, 256 + 8 * lane, wt);
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
  for (int base = first; base < p.h_q; base += kBatch * step) {
    if (base != first) load(base);
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (base + i * step >= p.h_q) break;
      const int h = base + i * step + (lane >> 3);
      float x[8];
      unpack8(raw[i], x);
      rotate<MODE>(x, ang, kRot, l, true);
      if (h < p.h_q)
        *reinterpret_cast<uint4*>(p.q_out + t * p.qo_tok + h * p.qo_head + 8 * l) = pack8(x);
    }
  }
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Warps that fill the GPU once at half occupancy: with fewer, a token's heads
// are spread over more warps.
constexpr long long kFillWarps = 148 * 32;

int pick_split(int rows, int most) {
  long long n = (kFillWarps + rows - 1) / rows;
  if (n > most) n = most;
  return n < 1 ? 1 : static_cast<int>(n);
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
  p.Hq = q.data ? Hq : 0;
  p.Hkv = Hkv;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.zero_skipped = zero_skipped;
  p.nsplit = pick_split(p.tk.rows, (p.Hq + 2 * Hkv + 1) / 2);
  const long long warps = static_cast<long long>(p.tk.rows) * p.nsplit;
  const long long grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > INT_MAX) return cudaErrorInvalidValue;
  const int g = static_cast<int>(grid);
  if (group) {
    if (mode == kNoRope) kv_append_gqa_kernel<kNoRope, true><<<g, kThreads, 0, stream>>>(p, group);
    else if (mode == kHalves) kv_append_gqa_kernel<kHalves, true><<<g, kThreads, 0, stream>>>(p, group);
    else kv_append_gqa_kernel<kPairs, true><<<g, kThreads, 0, stream>>>(p, group);
  } else {
    if (mode == kNoRope) kv_append_gqa_kernel<kNoRope, false><<<g, kThreads, 0, stream>>>(p, 0);
    else if (mode == kHalves) kv_append_gqa_kernel<kHalves, false><<<g, kThreads, 0, stream>>>(p, 0);
    else kv_append_gqa_kernel<kPairs, false><<<g, kThreads, 0, stream>>>(p, 0);
  }
  return cudaGetLastError();
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
  const int g = static_cast<int>(grid);
  if (mode == kNoRope) kv_append_mla_kernel<kNoRope><<<g, kThreads, 0, stream>>>(p);
  else if (mode == kHalves) kv_append_mla_kernel<kHalves><<<g, kThreads, 0, stream>>>(p);
  else kv_append_mla_kernel<kPairs><<<g, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
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
