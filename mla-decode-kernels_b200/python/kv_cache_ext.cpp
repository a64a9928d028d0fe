// PyTorch binding of include/kv_append.h and include/kv4_decode.h: tensor
// checks, then the C entry points on the current torch stream.  Compiled into
// the same module as gqa_decode_ext.cpp, which calls bind_kv_cache.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cstdlib>
#include <tuple>

#include "kv4_decode.h"
#include "kv_append.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

void check_status(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e));
}

int as_int(int64_t v, const char* name) {
  TORCH_CHECK(v >= 0 && v <= INT_MAX, name, " is out of range");
  return static_cast<int>(v);
}

void check_i32(const torch::Tensor& t, const torch::Device& dev, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, name, " must be a CUDA tensor on the cache's device");
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.is_contiguous(), name,
              " must be contiguous int32");
}

bool aligned16(const torch::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

void check_cache(const torch::Tensor& t, torch::ScalarType type, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", c10::toString(type));
  TORCH_CHECK(t.dim() == 4 && t.is_contiguous() && aligned16(t), name,
              " must be a contiguous, 16-byte aligned tensor of four dims");
  TORCH_CHECK(t.numel() > 0, name, " must not be empty");
}

// Rows of heads [rows, heads, dim] (or [rows, dim]) that may be strided views,
// e.g. slices of one projection's output: the last dim contiguous, the others
// in steps of 8 elements, 16-byte aligned.
void check_rows(const torch::Tensor& t, const torch::Device& dev, int64_t dim, int dims,
                const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, name, " must be a CUDA tensor on the cache's device");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.dim() == dims && t.size(dims - 1) == dim, name, " must have ", dims,
              " dims, the last of size ", dim);
  TORCH_CHECK(t.stride(dims - 1) == 1, name, "'s last dim must be contiguous");
  if (t.numel() == 0) return;
  TORCH_CHECK(aligned16(t), name, " must be 16-byte aligned");
  for (int d = 0; d + 1 < dims; ++d)
    TORCH_CHECK(t.size(d) == 1 || t.stride(d) % 8 == 0, name,
                "'s strides must be multiples of 8 elements");
}

// A stride that is never used (size 1) may be anything; the kernels want
// multiples of 8.
long long used_stride(const torch::Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }

kv_append_heads heads(const torch::Tensor& t, bool with_heads) {
  return {reinterpret_cast<const gqa_bf16*>(t.data_ptr()), used_stride(t, 0),
          with_heads ? used_stride(t, 1) : 0};
}

kv_append_norm norm(const OptTensor& w, const torch::Device& dev, int64_t dim, double eps,
                    const char* name) {
  if (!w) return {nullptr, 0, 0.f};
  TORCH_CHECK(w->is_cuda() && w->device() == dev, name,
              " must be a CUDA tensor on the cache's device");
  TORCH_CHECK(w->scalar_type() == torch::kBFloat16 || w->scalar_type() == torch::kFloat32, name,
              " must be bf16 or fp32");
  TORCH_CHECK(w->dim() == 1 && w->size(0) == dim && w->is_contiguous() && aligned16(*w), name,
              " must be a contiguous, 16-byte aligned [", dim, "] tensor");
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  return {w->data_ptr(), w->scalar_type() == torch::kFloat32 ? 1 : 0, static_cast<float>(eps)};
}

kv_append_rope rope(const OptTensor& table, const torch::Device& dev, bool interleaved) {
  if (!table) return {nullptr, 0, 0, 0};
  TORCH_CHECK(table->is_cuda() && table->device() == dev,
              "cos_sin must be a CUDA tensor on the cache's device");
  TORCH_CHECK(table->scalar_type() == torch::kFloat32 && table->dim() == 2 &&
                  table->is_contiguous() && aligned16(*table),
              "cos_sin must be a contiguous, 16-byte aligned fp32 [positions, rotary_dim] tensor");
  TORCH_CHECK(table->size(0) >= 1, "cos_sin must hold a position");
  return {table->data_ptr<float>(), as_int(table->size(1), "rotary_dim"),
          as_int(table->size(0), "positions of cos_sin"), interleaved ? 1 : 0};
}

kv_append_tokens tokens(int64_t rows, const torch::Tensor& block_table,
                        const torch::Tensor& seq_lens, const OptTensor& cu_seqlens,
                        const OptTensor& positions, int64_t num_blocks, int64_t block_size,
                        const torch::Device& dev) {
  check_i32(block_table, dev, "block_table");
  check_i32(seq_lens, dev, "seq_lens");
  TORCH_CHECK(seq_lens.dim() == 1, "seq_lens must be [B]");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == seq_lens.size(0) &&
                  block_table.size(1) >= 1,
              "block_table must be [B, max_blocks]");
  if (cu_seqlens) {
    check_i32(*cu_seqlens, dev, "cu_seqlens");
    TORCH_CHECK(cu_seqlens->dim() == 1 && cu_seqlens->size(0) == seq_lens.size(0) + 1,
                "cu_seqlens must be [B + 1]");
  } else {
    TORCH_CHECK(rows == seq_lens.size(0), "without cu_seqlens there is one row per request");
  }
  if (positions) {
    check_i32(*positions, dev, "positions");
    TORCH_CHECK(positions->dim() == 1 && positions->size(0) == rows, "positions must be [rows]");
  }
  return {block_table.data_ptr<int>(),
          seq_lens.data_ptr<int>(),
          cu_seqlens ? cu_seqlens->data_ptr<int>() : nullptr,
          positions ? positions->data_ptr<int>() : nullptr,
          as_int(rows, "rows"),
          as_int(seq_lens.size(0), "batch"),
          as_int(block_table.size(1), "max_blocks"),
          as_int(num_blocks, "num_blocks"),
          as_int(block_size, "block_size")};
}

// Dim-group size of a 4-bit cache [num_blocks, block_size / 16, Hkv, tile].
int kv4_group(const torch::Tensor& k_cache, const torch::Tensor& v_cache) {
  check_cache(k_cache, torch::kUInt8, "k_cache");
  check_cache(v_cache, torch::kUInt8, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.device() == v_cache.device(),
              "k_cache and v_cache must have the same shape and device");
  for (int group : {32, 64, 128})
    if (k_cache.size(3) == static_cast<int64_t>(kv4_tile_bytes(group))) return group;
  TORCH_CHECK(false, "the last dim of a 4-bit cache must be 1280, 1152 or 1088 (group 32, 64, 128)");
}

// Refuses overlaps that show from the tensors' bounds: of two views of one
// buffer whose rows interleave nothing is said.
void apart(const torch::Tensor& a, const torch::Tensor& b, const char* an, const char* bn) {
  const auto o = at::get_overlap_status(a, b);
  TORCH_CHECK(o != at::MemOverlapStatus::Full && o != at::MemOverlapStatus::Partial, an,
              " must not overlap ", bn);
}

// Whether rows of heads a and b [rows, heads, dim] of equal strides, as slices
// of one projection have, share memory; with a itself: whether two of its
// heads do.  Head (t, h) of a and (t', h') of b are delta + dt ts + dh hs
// elements apart, and share memory where that is less than dim.
bool rows_meet(const torch::Tensor& a, const torch::Tensor& b) {
  const int64_t T = a.size(0), dim = a.size(2), ts = used_stride(a, 0);
  const int64_t hs = a.size(1) > 1 ? a.stride(1) : used_stride(b, 1);
  const int64_t delta = (reinterpret_cast<intptr_t>(b.data_ptr()) -
                         reinterpret_cast<intptr_t>(a.data_ptr())) / a.element_size();
  const bool self = a.is_same(b);
  for (int64_t dh = 1 - a.size(1); dh < b.size(1); ++dh) {
    const int64_t at = delta + dh * hs;
    // the closest is this dt or one next to it
    const int64_t near = ts > 0 ? std::clamp(-at / ts, 1 - T, T - 1) : 0;
    for (int64_t dt = std::max(near - 1, 1 - T); dt <= std::min(near + 1, T - 1); ++dt)
      if (!(self && dt == 0 && dh == 0) && std::abs(at + dt * ts) < dim) return true;
  }
  return false;
}

// apart() for an output and an input of rows of heads, exact where their
// strides are equal.
void rows_apart(const torch::Tensor& a, const torch::Tensor& b, const char* an, const char* bn) {
  if (a.numel() == 0 || b.numel() == 0) return;
  if (used_stride(a, 0) == used_stride(b, 0) &&
      (a.size(1) == 1 || b.size(1) == 1 || a.stride(1) == b.stride(1))) {
    TORCH_CHECK(!rows_meet(a, b), an, " must not overlap ", bn);
  } else {
    apart(a, b, an, bn);
  }
}

// The output of a rotated q: `out` after checks, or a new tensor.
torch::Tensor rotated_out(const torch::Tensor& q, const OptTensor& out, const torch::Device& dev) {
  if (!out) return torch::empty(q.sizes(), q.options());
  check_rows(*out, dev, q.size(2), 3, "out");
  TORCH_CHECK(out->sizes() == q.sizes(), "out must have q's shape");
  TORCH_CHECK(out->numel() == 0 || !rows_meet(*out, *out), "out's elements must not share memory");
  // Every element is read and written by one thread, so q's own place is fine.
  if (out->numel() > 0 && out->data_ptr() == q.data_ptr()) {
    TORCH_CHECK(used_stride(*out, 0) == used_stride(q, 0) &&
                    used_stride(*out, 1) == used_stride(q, 1),
                "out may be q, but not another view of its memory");
  } else {
    rows_apart(*out, q, "out", "q");
  }
  return *out;
}

OptTensor gqa_append(OptTensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                     torch::Tensor v_cache, torch::Tensor block_table, torch::Tensor seq_lens,
                     OptTensor cos_sin, OptTensor cu_seqlens, OptTensor positions,
                     bool interleaved, OptTensor q_weight, OptTensor k_weight, double eps,
                     OptTensor out, bool kv4) {
  int group = 0;
  if (kv4) {
    group = kv4_group(k_cache, v_cache);
  } else {
    check_cache(k_cache, torch::kBFloat16, "k_cache");
    check_cache(v_cache, torch::kBFloat16, "v_cache");
    TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.device() == v_cache.device(),
                "k_cache and v_cache must have the same shape and device");
    TORCH_CHECK(k_cache.size(3) == 128, "k_cache must be [num_blocks, block_size, Hkv, 128]");
  }
  apart(k_cache, v_cache, "k_cache", "v_cache");
  const torch::Device dev = k_cache.device();
  const int64_t block_size = kv4 ? 16 * k_cache.size(1) : k_cache.size(1);
  const int64_t Hkv = k_cache.size(2);
  check_rows(k, dev, 128, 3, "k");
  check_rows(v, dev, 128, 3, "v");
  TORCH_CHECK(k.size(1) == Hkv && v.sizes() == k.sizes(), "k and v must be [rows, Hkv, 128]");
  const int64_t rows = k.size(0);
  if (q) {
    check_rows(*q, dev, 128, 3, "q");
    TORCH_CHECK(q->size(0) == rows, "q, k and v must have the same rows");
    TORCH_CHECK(q->size(1) >= 1, "q must have a head");
  } else {
    TORCH_CHECK(!out && !q_weight, "out and q_weight need q");
  }
  const kv_append_tokens tk = tokens(rows, block_table, seq_lens, cu_seqlens, positions,
                                     k_cache.size(0), block_size, dev);
  const kv_append_rope rp = rope(cos_sin, dev, interleaved);
  TORCH_CHECK(!cos_sin || (rp.rotary_dim >= 16 && rp.rotary_dim <= 128 && rp.rotary_dim % 16 == 0),
              "rotary_dim must be a multiple of 16 up to 128");
  const kv_append_norm qn = norm(q_weight, dev, 128, eps, "q_weight");
  const kv_append_norm kn = norm(k_weight, dev, 128, eps, "k_weight");
  const c10::cuda::CUDAGuard guard(dev);
  OptTensor result;
  kv_append_heads qh{nullptr, 0, 0};
  long long out_tok = 0, out_head = 0;
  if (q) {
    result = rotated_out(*q, out, dev);
    if (out) {
      rows_apart(*out, k, "out", "k");
      rows_apart(*out, v, "out", "v");
      apart(*out, k_cache, "out", "k_cache");
      apart(*out, v_cache, "out", "v_cache");
    }
    if (rows) qh = heads(*q, true);
    out_tok = used_stride(*result, 0);
    out_head = used_stride(*result, 1);
  }
  if (rows == 0) return result;
  gqa_bf16* qo = q ? reinterpret_cast<gqa_bf16*>(result->data_ptr()) : nullptr;
  const int Hq = q ? as_int(q->size(1), "Hq") : 0, hkv = as_int(Hkv, "Hkv");
  const int zero = out ? 0 : 1;
  const auto stream = at::cuda::getCurrentCUDAStream();
  if (kv4)
    check_status(kv_append_gqa_kv4_launch(&tk, &rp, qh, heads(k, true), heads(v, true), qn, kn, qo,
                                          out_tok, out_head, zero, k_cache.data_ptr<uint8_t>(),
                                          v_cache.data_ptr<uint8_t>(), Hq, hkv, group, stream),
                 "gqa_append_kv4");
  else
    check_status(kv_append_gqa_launch(&tk, &rp, qh, heads(k, true), heads(v, true), qn, kn, qo,
                                      out_tok, out_head, zero,
                                      reinterpret_cast<gqa_bf16*>(k_cache.data_ptr()),
                                      reinterpret_cast<gqa_bf16*>(v_cache.data_ptr()), Hq, hkv,
                                      stream),
                 "gqa_append");
  return result;
}

OptTensor mla_append(torch::Tensor kv_c, torch::Tensor k_pe, torch::Tensor kv_cache,
                     torch::Tensor block_table, torch::Tensor seq_lens, OptTensor cos_sin,
                     OptTensor q_pe, OptTensor cu_seqlens, OptTensor positions, bool interleaved,
                     OptTensor kv_weight, double eps, OptTensor out) {
  check_cache(kv_cache, torch::kBFloat16, "kv_cache");
  TORCH_CHECK(kv_cache.size(1) == 64 && kv_cache.size(2) == 1 && kv_cache.size(3) == 576,
              "kv_cache must be [num_blocks, 64, 1, 576]");
  const torch::Device dev = kv_cache.device();
  check_rows(kv_c, dev, 512, 2, "kv_c");
  check_rows(k_pe, dev, 64, 2, "k_pe");
  const int64_t rows = kv_c.size(0);
  TORCH_CHECK(k_pe.size(0) == rows, "kv_c and k_pe must have the same rows");
  if (q_pe) {
    check_rows(*q_pe, dev, 64, 3, "q_pe");
    TORCH_CHECK(q_pe->size(0) == rows, "q_pe, kv_c and k_pe must have the same rows");
    TORCH_CHECK(q_pe->size(1) >= 1, "q_pe must have a head");
  } else {
    TORCH_CHECK(!out, "out needs q_pe");
  }
  const kv_append_tokens tk = tokens(rows, block_table, seq_lens, cu_seqlens, positions,
                                     kv_cache.size(0), 64, dev);
  const kv_append_rope rp = rope(cos_sin, dev, interleaved);
  TORCH_CHECK(!cos_sin || rp.rotary_dim == 64, "cos_sin must be [positions, 64]");
  const kv_append_norm nm = norm(kv_weight, dev, 512, eps, "kv_weight");
  const c10::cuda::CUDAGuard guard(dev);
  OptTensor result;
  kv_append_heads qh{nullptr, 0, 0};
  long long out_tok = 0, out_head = 0;
  if (q_pe) {
    result = rotated_out(*q_pe, out, dev);
    if (out) {
      apart(*out, kv_c, "out", "kv_c");
      apart(*out, k_pe, "out", "k_pe");
      apart(*out, kv_cache, "out", "kv_cache");
    }
    if (rows) qh = heads(*q_pe, true);
    out_tok = used_stride(*result, 0);
    out_head = used_stride(*result, 1);
  }
  if (rows == 0) return result;
  check_status(kv_append_mla_launch(&tk, &rp, heads(kv_c, false), heads(k_pe, false), nm, qh,
                                    q_pe ? reinterpret_cast<gqa_bf16*>(result->data_ptr()) : nullptr,
                                    out_tok, out_head, out ? 0 : 1,
                                    reinterpret_cast<gqa_bf16*>(kv_cache.data_ptr()),
                                    q_pe ? as_int(q_pe->size(1), "h_q") : 0,
                                    at::cuda::getCurrentCUDAStream()),
               "mla_append");
  return result;
}

torch::Tensor gqa_decode_kv4(torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache,
                             torch::Tensor block_table, torch::Tensor seq_lens, double scale,
                             OptTensor out) {
  const int group = kv4_group(k_cache, v_cache);
  const torch::Device dev = k_cache.device();
  TORCH_CHECK(q.is_cuda() && q.device() == dev, "q must be a CUDA tensor on the cache's device");
  TORCH_CHECK(q.scalar_type() == torch::kBFloat16, "q must be bf16");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && q.is_contiguous(),
              "q must be a contiguous [B, Hq, 128] tensor");
  const int64_t B = q.size(0), Hq = q.size(1), Hkv = k_cache.size(2);
  TORCH_CHECK(Hq >= 1 && Hq % Hkv == 0, "Hq must be divisible by Hkv");
  TORCH_CHECK(Hq / Hkv <= 128, "Hq / Hkv must be at most 128");
  check_i32(block_table, dev, "block_table");
  check_i32(seq_lens, dev, "seq_lens");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == B && block_table.size(1) >= 1,
              "block_table must be [B, max_blocks]");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == B, "seq_lens must be [B]");
  if (out) {
    TORCH_CHECK(out->is_cuda() && out->device() == dev && out->scalar_type() == torch::kBFloat16 &&
                    out->is_contiguous() && out->sizes() == q.sizes(),
                "out must be a contiguous bf16 tensor of q's shape on the cache's device");
    apart(*out, q, "out", "q");
    apart(*out, k_cache, "out", "k_cache");
    apart(*out, v_cache, "out", "v_cache");
  }
  const c10::cuda::CUDAGuard guard(dev);
  torch::Tensor o = out ? *out : torch::empty_like(q);
  if (B == 0) return o;
  TORCH_CHECK(aligned16(q) && aligned16(o), "q and out must be 16-byte aligned");
  const int b = as_int(B, "B"), hq = as_int(Hq, "Hq"), hkv = as_int(Hkv, "Hkv");
  const size_t bytes = kv4_decode_workspace_bytes(b, hq, hkv, group);
  TORCH_CHECK(bytes > 0, "gqa_decode_kv4: no workspace size for these dims");
  // From the caching allocator on the current stream, for this call alone: two
  // streams, threads or captured graphs never share one.
  torch::Tensor ws = torch::empty({static_cast<int64_t>(bytes)}, k_cache.options());
  check_status(kv4_decode_launch(reinterpret_cast<const gqa_bf16*>(q.data_ptr()),
                                 k_cache.data_ptr<uint8_t>(), v_cache.data_ptr<uint8_t>(),
                                 block_table.data_ptr<int>(), seq_lens.data_ptr<int>(),
                                 reinterpret_cast<gqa_bf16*>(o.data_ptr()), b, hq, hkv, group,
                                 as_int(16 * k_cache.size(1), "block_size"),
                                 as_int(block_table.size(1), "max_blocks"),
                                 as_int(k_cache.size(0), "num_blocks"), static_cast<float>(scale),
                                 ws.data_ptr(), bytes, at::cuda::getCurrentCUDAStream()),
               "gqa_decode_kv4");
  return o;
}

std::tuple<torch::Tensor, torch::Tensor> gqa_gather_kv4(torch::Tensor k_cache,
                                                        torch::Tensor v_cache,
                                                        torch::Tensor block_table,
                                                        torch::Tensor seq_lens,
                                                        OptTensor cu_seqlens, int64_t rows) {
  const int group = kv4_group(k_cache, v_cache);
  const torch::Device dev = k_cache.device();
  TORCH_CHECK(rows >= 0, "rows must not be negative");
  const kv_append_tokens tk = tokens(rows, block_table, seq_lens, cu_seqlens, c10::nullopt,
                                     k_cache.size(0), 16 * k_cache.size(1), dev);
  const c10::cuda::CUDAGuard guard(dev);
  const auto opts = k_cache.options().dtype(torch::kBFloat16);
  auto k = torch::empty({rows, k_cache.size(2), 128}, opts);
  auto v = torch::empty({rows, k_cache.size(2), 128}, opts);
  if (rows == 0) return {k, v};
  check_status(kv4_gather_launch(k_cache.data_ptr<uint8_t>(), v_cache.data_ptr<uint8_t>(),
                                 tk.block_table, tk.seq_lens, tk.cu_seqlens,
                                 reinterpret_cast<gqa_bf16*>(k.data_ptr()),
                                 reinterpret_cast<gqa_bf16*>(v.data_ptr()), tk.rows, tk.batch,
                                 as_int(k_cache.size(2), "Hkv"), group, tk.block_size,
                                 tk.max_blocks, tk.num_blocks, at::cuda::getCurrentCUDAStream()),
               "gqa_gather_kv4");
  return {k, v};
}

int64_t status_of(int v, const char* what) {
  TORCH_CHECK(v >= 0, what, ": reading the status word failed");
  return v;
}

}  // namespace

void bind_kv_cache(pybind11::module_& m) {
  m.def("gqa_append", &gqa_append, "head norm, rotation and paged append of K and V");
  m.def("mla_append", &mla_append, "latent norm, rotation and append to the latent cache");
  m.def("gqa_decode_kv4", &gqa_decode_kv4, "GQA decode over a 4-bit paged cache");
  m.def("gqa_gather_kv4", &gqa_gather_kv4, "tokens of a 4-bit paged cache as bf16");
  m.def("kv4_tile_bytes", [](int64_t group) {
    return static_cast<int64_t>(kv4_tile_bytes(static_cast<int>(group)));
  });
  m.def("kv_append_get_status",
        [](bool clear) { return status_of(kv_append_get_status(clear ? 1 : 0), "kv_append"); },
        py::arg("clear") = false);
  m.def("kv4_get_status",
        [](bool clear) { return status_of(kv4_decode_get_status(clear ? 1 : 0), "kv4_decode"); },
        py::arg("clear") = false);
}
