// Torch-side entry of the 4-bit cache operators: argument checks, outputs and workspaces from torch's
// stream-ordered allocator, the current stream, and the call through the C ABI.
//
// The other operators do this in Python over ctypes. A decode step makes one write and one attention call a
// layer, each a few microseconds of GPU time, and the Python form of these checks took 60 to 90 us a call on
// the host; here it is a few. libw4a8.so stays free of torch: this module gets the addresses of its
// entry points from int4_int8_ext (set_library).
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>

#include "w4a8.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

decltype(&w4a8_kv_write_int4) g_write;
decltype(&w4a8_kv_read_int4) g_read;
decltype(&w4a8_attention_int4) g_attend;
decltype(&w4a8_attention_int4_workspace) g_workspace;

void set_library(uintptr_t write, uintptr_t read, uintptr_t attend, uintptr_t workspace) {
  g_write = reinterpret_cast<decltype(g_write)>(write);
  g_read = reinterpret_cast<decltype(g_read)>(read);
  g_attend = reinterpret_cast<decltype(g_attend)>(attend);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(workspace);
}

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }
inline void require(bool ok, const char* what) {
  if (!ok) fail(what);
}
inline void require(bool ok, const char* name, const char* what) {
  if (!ok) fail(std::string(name) + what);
}
void check(int rc, const char* what) {
  if (!rc) return;
  const char* text = rc == W4A8_ERR_ARG           ? "invalid argument"
                     : rc == W4A8_ERR_ALIGN       ? "alignment (pointer or stride not 16-byte aligned)"
                     : rc == W4A8_ERR_UNSUPPORTED ? "unsupported geometry"
                     : rc == W4A8_ERR_LAUNCH      ? "CUDA launch error"
                                                  : "unknown";
  fail(std::string(what) + " failed: libw4a8 status " + std::to_string(rc) + " (" + text + ")");
}

// w4a8 number of a torch type; -1 for one that rows cannot have.
int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? W4A8_F32 : t == at::kHalf ? W4A8_F16 : t == at::kBFloat16 ? W4A8_BF16 : -1;
}
at::ScalarType type_of(int dtype) {
  return dtype == W4A8_F32 ? at::kFloat : dtype == W4A8_F16 ? at::kHalf : at::kBFloat16;
}

void check_index(const Tensor& t, const char* name, int dim, const Tensor& like) {
  require(t.scalar_type() == at::kInt, name, " must be int32");
  if (t.dim() != dim) fail(std::string(name) + " must be rank-" + std::to_string(dim));
  require(t.device() == like.device(), name, " must be on the cache's device");
  require(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have a contiguous last dimension");
}

void check_constant(const Tensor& t, const char* name) {
  require(!(t.requires_grad() && c10::GradMode::is_enabled()), name,
          " requires a gradient, which the 4-bit cache does not have: use torch.no_grad()");
  require(!t._fw_grad(0).defined(), name, " has a forward-mode tangent, which the 4-bit cache does not carry");
}

void check_rows(const Tensor& t, const char* name, int64_t heads, const Tensor& k_codes) {
  require(t.device() == k_codes.device(), name, " must be on the cache's device");
  require(t.dim() == 3, name, " must be rank-3 [rows, heads, head_dim]");
  require(dtype_of(t.scalar_type()) >= 0, name, " must be float32, float16 or bfloat16");
  require(t.size(2) == 2 * k_codes.size(3), name, " must have the cache's head_dim");
  require(heads < 0 || t.size(1) == heads, name, " must have the cache's heads");
  require(t.numel() == 0 || t.stride(2) == 1, name, " must have a contiguous last dimension");
  check_constant(t, name);
}

void check_codes(const Tensor& k_codes) {
  require(k_codes.dim() == 4, "k_codes must be rank-4 [pages, kv_heads, page_size, head_dim / 2]");
}

w4a8_kv_cache make_cache(const Tensor& k_codes, const Tensor& v_codes, const Tensor& scales, const Tensor& block_table,
                         const Tensor& seq_lens, const OptTensor& cu_q, int64_t rows) {
  constexpr int64_t kMost = 0x7fffffff;
  check_codes(k_codes);
  require(k_codes.scalar_type() == at::kByte && v_codes.scalar_type() == at::kByte,
          "k_codes and v_codes must be uint8");
  require(k_codes.sizes() == v_codes.sizes() && k_codes.strides() == v_codes.strides(),
          "k_codes and v_codes must have the same shape and strides");
  require(v_codes.device() == k_codes.device() && scales.device() == k_codes.device(),
          "the cache's tensors must be on one device");
  const int64_t pages = k_codes.size(0), heads = k_codes.size(1), page_size = k_codes.size(2), d = 2 * k_codes.size(3);
  require(d == 64 || d == 96 || d == 128 || d == 192 || d == 256, "head_dim must be 64, 96, 128, 192 or 256");
  require(heads >= 1 && page_size >= 1, "the cache must have heads and rows in a page");
  require(scales.dim() == 5 && scales.size(0) == pages && scales.size(1) == heads && scales.size(2) == page_size &&
              scales.size(3) == 2,
          "scales must be rank-5 [pages, kv_heads, page_size, 2, head_dim / group]");
  require(scales.scalar_type() == at::kBFloat16, "scales must be bfloat16");
  check_constant(scales, "scales");
  const int64_t groups = scales.size(4);
  require(groups > 0 && (32 * groups == d || 64 * groups == d || 128 * groups == d),
          "scales must hold one value for 32, 64 or 128 channels");
  require(pages == 0 ||
              (k_codes.stride(3) == 1 && scales.stride(3) == groups && (groups == 1 || scales.stride(4) == 1)),
          "rows of the cache must be contiguous");
  check_index(block_table, "block_table", 2, k_codes);
  check_index(seq_lens, "seq_lens", 1, k_codes);
  const int64_t batch = seq_lens.size(0);
  require(block_table.size(0) == batch, "block_table must have a row for each sequence");
  require(rows <= kMost && pages <= kMost && page_size <= kMost && block_table.size(1) <= kMost && heads <= kMost &&
              batch <= kMost,
          "sizes must fit 32 bits");
  require(block_table.size(1) * page_size <= (int64_t(1) << 30), "a row of block_table must name at most 2^30 tokens");
  if (cu_q) {
    check_index(*cu_q, "cu_q", 1, k_codes);
    require(cu_q->size(0) == batch + 1, "cu_q must be [batch + 1]");
  } else {
    require(batch > 0 || rows == 0, "rows without a sequence need cu_q");
    require(batch == 0 || rows % batch == 0, "without cu_q every sequence has the same number of rows");
  }
  require(k_codes.is_cuda(), "k_codes must be a CUDA tensor");
  w4a8_kv_cache c;
  c.k_codes = static_cast<uint8_t*>(k_codes.data_ptr());
  c.v_codes = static_cast<uint8_t*>(v_codes.data_ptr());
  c.scales = scales.data_ptr();
  c.code_page = k_codes.stride(0), c.code_head = k_codes.stride(1), c.code_tok = k_codes.stride(2);
  c.scale_page = scales.stride(0), c.scale_head = scales.stride(1), c.scale_tok = scales.stride(2);
  c.pages = int(pages), c.page_size = int(page_size), c.heads = int(heads);
  c.head_dim = int(d), c.group = int(d / groups);
  c.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  c.table_ld = block_table.stride(0);
  c.table_cols = int(block_table.size(1));
  c.batch = int(batch);
  c.seq_lens = static_cast<const int32_t*>(seq_lens.data_ptr());
  c.cu_q = cu_q ? static_cast<const int32_t*>(cu_q->data_ptr()) : nullptr;
  c.rows = int(rows);
  return c;
}

void* current_stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

const float* step_of(const OptTensor& step, const char* name, const w4a8_kv_cache& c, const Tensor& k_codes) {
  if (!step) return nullptr;
  require(step->is_contiguous(), name, " must be contiguous");
  require(step->scalar_type() == at::kFloat && step->device() == k_codes.device() && step->dim() == 2 &&
              step->size(0) == c.heads && step->size(1) == c.head_dim / c.group,
          name, " must be float32 [kv_heads, head_dim / group] on the cache's device");
  return static_cast<const float*>(step->data_ptr());
}

void kv_write(const Tensor& k, const Tensor& v, const Tensor& k_codes, const Tensor& v_codes, const Tensor& scales,
              const Tensor& block_table, const Tensor& seq_lens, const OptTensor& cu_q, const OptTensor& k_step,
              const OptTensor& v_step) {
  check_codes(k_codes);
  check_rows(k, "k", k_codes.size(1), k_codes);
  check_rows(v, "v", k_codes.size(1), k_codes);
  if (k_step) check_constant(*k_step, "k_step");
  if (v_step) check_constant(*v_step, "v_step");
  require(v.size(0) == k.size(0) && v.scalar_type() == k.scalar_type(), "k and v must have the same shape and type");
  const int64_t rows = k.size(0);
  const w4a8_kv_cache c = make_cache(k_codes, v_codes, scales, block_table, seq_lens, cu_q, rows);
  const float* ks = step_of(k_step, "k_step", c, k_codes);
  const float* vs = step_of(v_step, "v_step", c, k_codes);
  if (!rows) return;
  const c10::cuda::CUDAGuard guard(k.device());
  check(g_write(&c, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                dtype_of(k.scalar_type()), ks, vs, current_stream(k)),
        "w4a8_kv_write_int4");
}

std::tuple<Tensor, Tensor> kv_read(const Tensor& k_codes, const Tensor& v_codes, const Tensor& scales,
                                   const Tensor& block_table, const Tensor& seq_lens, const OptTensor& cu_q,
                                   int64_t rows, int dtype) {
  require(rows >= 0, "rows must not be negative");
  const w4a8_kv_cache c = make_cache(k_codes, v_codes, scales, block_table, seq_lens, cu_q, rows);
  const auto options = k_codes.options().dtype(type_of(dtype));
  const int64_t shape[3] = {rows, c.heads, c.head_dim};
  const c10::cuda::CUDAGuard guard(k_codes.device());
  if (c.batch == 0) return {at::zeros(shape, options), at::zeros(shape, options)};
  Tensor k = at::empty(shape, options), v = at::empty(shape, options);
  if (rows) check(g_read(&c, k.data_ptr(), v.data_ptr(), dtype, current_stream(k_codes)), "w4a8_kv_read_int4");
  return {k, v};
}

std::tuple<Tensor, OptTensor> attend(const Tensor& q, const Tensor& k_codes, const Tensor& v_codes,
                                     const Tensor& scales, const Tensor& block_table, const Tensor& seq_lens,
                                     const OptTensor& cu_q, std::optional<int64_t> max_q,
                                     std::optional<int64_t> max_len, bool causal, int64_t window,
                                     std::optional<double> scale, bool with_lse) {
  check_codes(k_codes);
  check_rows(q, "q", -1, k_codes);
  const int64_t rows = q.size(0), q_heads = q.size(1), kv_heads = k_codes.size(1);
  require(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0, "q_heads must be a multiple of kv_heads");
  require(q_heads <= 0x7fffffff, "sizes must fit 32 bits");
  require(window >= 0 && window <= 0x7fffffff, "window must not be negative and must fit 32 bits");
  const w4a8_kv_cache c = make_cache(k_codes, v_codes, scales, block_table, seq_lens, cu_q, rows);
  int64_t most = c.batch ? rows / c.batch : 0;
  if (cu_q) {
    most = max_q ? std::min(*max_q, rows) : rows;
    require(most >= 1 || rows == 0, "max_q must be positive");
  } else {
    require(!max_q || *max_q >= most, "max_q must not be below the rows of a sequence");
  }
  int64_t len = int64_t(c.table_cols) * c.page_size;
  if (max_len) len = std::min(*max_len, len);
  require(len >= 0, "max_len must not be negative");
  const int dtype = dtype_of(q.scalar_type());
  const c10::cuda::CUDAGuard guard(q.device());
  if (c.batch == 0) {
    OptTensor lse;
    if (with_lse) lse = at::full({rows, q_heads}, -INFINITY, q.options().dtype(at::kFloat));
    return {at::zeros(q.sizes(), q.options()), lse};
  }
  Tensor out = at::empty(q.sizes(), q.options());
  OptTensor lse;
  if (with_lse) lse = at::empty({rows, q_heads}, q.options().dtype(at::kFloat));
  if (rows) {
    size_t bytes = 0;
    check(g_workspace(&c, int(q_heads), dtype, int(most), int(len), int(window), &bytes),
          "w4a8_attention_int4_workspace");
    Tensor workspace;  // released to the allocator after this call, in stream order
    if (bytes) workspace = at::empty({int64_t(bytes)}, k_codes.options());
    check(g_attend(&c, q.data_ptr(), q.stride(0), q.stride(1), int(q_heads), dtype, out.data_ptr(),
                   lse ? static_cast<float*>(lse->data_ptr()) : nullptr,
                   scale ? float(*scale) : float(1.0 / std::sqrt(double(c.head_dim))), causal, int(window), int(most),
                   int(len), bytes ? workspace.data_ptr() : nullptr, bytes, current_stream(q)),
          "w4a8_attention_int4");
  }
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("set_library", &set_library);
  m.def("kv_write", &kv_write);
  m.def("kv_read", &kv_read);
  m.def("attend", &attend);
}
