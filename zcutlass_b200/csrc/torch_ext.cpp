// PyTorch operator registration for the zcutlass GEMM (CUDA dispatch key only).
//
//   torch.ops.zcutlass_torch.gemm(A, B, C=None, bias=None, alpha=1.0, beta=0.0) -> D
//       same schema, checks and error behaviour as the reference op
//       (python/zcutlass_torch/csrc/zcutlass_torch.cpp:36-89, 153-156 in
//       supercatking/zcutlass): 2-D contiguous CUDA tensors, f16/bf16, D
//       allocated with at::empty, current CUDA stream, RuntimeError on failure.
//   torch.ops.zcutlass.gemm      the same op under the namespace the product spec names
//   torch.ops.zcutlass.gemm_out  writes into a caller-provided D (no allocation)
//   torch.ops.zcutlass.linear(x, weight, bias=None) -> y
//       nn.functional.linear semantics: weight is the PyTorch [N, K] layout and
//       is consumed directly as a column-major B (no transposed copy).
//   torch.ops.zcutlass.{quantize_fp8, gemm_fp8, linear_fp8, linear_fp8_out,
//       linear_fp8_train, rotary, rotary_}  8-bit block-scaled linears and
//       rotary positions over the C ABI (documented in torch_ops.py)
//
// This file only adapts tensors to the library's entry points; all kernels live in libzcutlass.so.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <optional>
#include <string_view>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "zcutlass/gemm.hpp"
#include "zcutlass_c.h"

namespace {

zcutlass::DType dtype_of(const at::Tensor& t) {
  if (t.scalar_type() == at::kHalf) return zcutlass::DType::F16;
  if (t.scalar_type() == at::kBFloat16) return zcutlass::DType::BF16;
  TORCH_CHECK(false, "zcutlass only supports float16 and bfloat16 tensors");
}

void check_2d_cuda_contiguous(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 2, name, " must be rank-2");
  TORCH_CHECK(t.is_contiguous(), name, " must be row-major contiguous");
  (void)dtype_of(t);
}

void check_operands(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>& c,
                    const std::optional<at::Tensor>& bias) {
  check_2d_cuda_contiguous(a, "A");
  check_2d_cuda_contiguous(b, "B");
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "A and B dtype must match");
  TORCH_CHECK(a.size(1) == b.size(0), "A.shape[1] must equal B.shape[0]");
  TORCH_CHECK(a.device() == b.device(), "A and B must be on the same CUDA device");
  if (c.has_value()) {
    check_2d_cuda_contiguous(*c, "C");
    TORCH_CHECK(c->scalar_type() == a.scalar_type(), "C dtype must match A/B");
    TORCH_CHECK(c->device() == a.device(), "C must be on the same CUDA device");
    TORCH_CHECK(c->size(0) == a.size(0) && c->size(1) == b.size(1),
                "C shape must be [A.shape[0], B.shape[1]]");
  }
  if (bias.has_value()) {
    TORCH_CHECK(bias->is_cuda(), "bias must be a CUDA tensor");
    TORCH_CHECK(bias->dim() == 1, "bias must be rank-1");
    TORCH_CHECK(bias->is_contiguous(), "bias must be contiguous");
    TORCH_CHECK(bias->scalar_type() == a.scalar_type(), "bias dtype must match A/B");
    TORCH_CHECK(bias->device() == a.device(), "bias must be on the same CUDA device");
    TORCH_CHECK(bias->size(0) == b.size(1), "bias length must equal B.shape[1]");
  }
}

void run_gemm(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>& c,
              const std::optional<at::Tensor>& bias, double alpha, double beta, at::Tensor& d) {
  const zcutlass::DType t = dtype_of(a);
  zcutlass::GemmDesc desc{a.size(0),
                          b.size(1),
                          a.size(1),
                          a.stride(0),
                          b.stride(0),
                          c.has_value() ? c->stride(0) : b.size(1),
                          d.stride(0),
                          t,
                          t,
                          t,
                          t,
                          static_cast<float>(alpha),
                          static_cast<float>(beta),
                          bias.has_value() ? bias->data_ptr() : nullptr,
                          at::cuda::getCurrentCUDAStream().stream()};
  const zcutlass::Status status = zcutlass::gemm(
      desc, a.data_ptr(), b.data_ptr(), c.has_value() ? c->data_ptr() : nullptr, d.data_ptr());
  TORCH_CHECK(status == zcutlass::Status::Success, "zcutlass::gemm failed: ",
              zcutlass::status_to_string(status));
}

at::Tensor gemm_op(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>& c,
                   const std::optional<at::Tensor>& bias, double alpha, double beta) {
  check_operands(a, b, c, bias);
  const c10::cuda::CUDAGuard guard(a.device());
  at::Tensor d = at::empty({a.size(0), b.size(1)}, a.options());
  run_gemm(a, b, c, bias, alpha, beta, d);
  return d;
}

void gemm_out_op(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>& c,
                 const std::optional<at::Tensor>& bias, double alpha, double beta, at::Tensor d) {
  check_operands(a, b, c, bias);
  check_2d_cuda_contiguous(d, "D");
  TORCH_CHECK(d.scalar_type() == a.scalar_type(), "D dtype must match A/B");
  TORCH_CHECK(d.device() == a.device(), "D must be on the same CUDA device");
  TORCH_CHECK(d.size(0) == a.size(0) && d.size(1) == b.size(1),
              "D shape must be [A.shape[0], B.shape[1]]");
  const c10::cuda::CUDAGuard guard(a.device());
  run_gemm(a, b, c, bias, alpha, beta, d);
}

// y[..., N] = x[..., K] @ weight[N, K]^T + bias
at::Tensor linear_op(const at::Tensor& x, const at::Tensor& weight,
                     const std::optional<at::Tensor>& bias) {
  TORCH_CHECK(x.is_cuda() && weight.is_cuda(), "x and weight must be CUDA tensors");
  TORCH_CHECK(weight.dim() == 2 && weight.is_contiguous(), "weight must be a contiguous [N, K] matrix");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == weight.size(1), "x.shape[-1] must equal weight.shape[1]");
  TORCH_CHECK(x.scalar_type() == weight.scalar_type(), "x and weight dtype must match");
  TORCH_CHECK(x.device() == weight.device(), "x and weight must be on the same CUDA device");
  const zcutlass::DType t = dtype_of(x);
  if (bias.has_value()) {
    TORCH_CHECK(bias->is_cuda() && bias->dim() == 1 && bias->is_contiguous(),
                "bias must be a contiguous rank-1 CUDA tensor");
    TORCH_CHECK(bias->scalar_type() == x.scalar_type(), "bias dtype must match x");
    TORCH_CHECK(bias->size(0) == weight.size(0), "bias length must equal weight.shape[0]");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor x2 = x.reshape({-1, x.size(-1)}).contiguous();
  const int64_t m = x2.size(0), k = x2.size(1), n = weight.size(0);
  std::vector<int64_t> out_shape(x.sizes().begin(), x.sizes().end());
  out_shape.back() = n;
  at::Tensor y = at::empty({m, n}, x.options());
  zcutlass::GemmDesc desc{m, n, k, x2.stride(0), weight.stride(0), n, n, t, t, t, t, 1.0f, 0.0f,
                          bias.has_value() ? bias->data_ptr() : nullptr,
                          at::cuda::getCurrentCUDAStream().stream()};
  desc.b_layout = zcutlass::layout::LayoutKind::ColumnMajor;
  const zcutlass::Status status =
      zcutlass::gemm(desc, x2.data_ptr(), weight.data_ptr(), nullptr, y.data_ptr());
  TORCH_CHECK(status == zcutlass::Status::Success, "zcutlass::linear failed: ",
              zcutlass::status_to_string(status));
  return y.view(out_shape);
}

// ---------------------------------------------------------------- 8-bit linears

void* current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_status(int status, const char* what) {
  TORCH_CHECK(status == ZCUTLASS_SUCCESS, what, " failed: ", zcutlass_status_to_string(status));
}

int32_t float_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kHalf: return ZCUTLASS_F16;
    case at::kBFloat16: return ZCUTLASS_BF16;
    case at::kFloat: return ZCUTLASS_F32;
    default: TORCH_CHECK(false, name, " must be float16, bfloat16 or float32");
  }
}

int32_t fp8_code(at::ScalarType t, const char* name) {
  TORCH_CHECK(t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2, name, " must be float8_e4m3fn or float8_e5m2");
  return t == at::kFloat8_e4m3fn ? ZCUTLASS_E4M3 : ZCUTLASS_E5M2;
}

constexpr int64_t kFp8Group = 128;
int64_t groups(int64_t n) { return (n + kFp8Group - 1) / kFp8Group; }

// Row stride of a matrix whose rows are contiguous (one row or no values: any; a multiple of 16 then).
int64_t row_stride(const at::Tensor& t, const char* name) {
  const int64_t any = (std::max<int64_t>(t.size(1), 1) + 15) / 16 * 16;
  if (t.numel() == 0) return any;
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have contiguous rows");
  if (t.size(0) == 1) return any;
  TORCH_CHECK(t.stride(0) >= t.size(1), name, " must not have overlapping rows");
  return t.stride(0);
}

// New tensors straight from the caching allocator: what these calls run on is often a few microseconds of
// kernel, so the dispatcher's share of at::empty and of the views after it would be most of the call.
at::Tensor empty_like_device(at::IntArrayRef sizes, at::ScalarType t, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, t, like.device(), std::nullopt));
}

// An 8-bit matrix with rows padded to 16 bytes (what TMA can describe).
at::Tensor empty_fp8(int64_t rows, int64_t cols, at::ScalarType t, const at::Tensor& like) {
  const int64_t ld = (cols + 15) / 16 * 16;
  at::Tensor q = empty_like_device({rows, ld}, t, like);
  q.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({rows, cols}), at::IntArrayRef({ld, int64_t(1)}));
  return q;
}

// Scales [rows, groups], rows contiguous: the product's kernels read the scales of neighbouring rows together.
at::Tensor empty_row_scales(int64_t rows, int64_t cols, const at::Tensor& like) {
  at::Tensor s = empty_like_device({groups(cols), rows}, at::kFloat, like);
  s.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({rows, groups(cols)}),
                                                 at::IntArrayRef({int64_t(1), std::max<int64_t>(rows, 1)}));
  return s;
}

struct Quantized {
  at::Tensor q, scale, qt, scale_t, col_sums;
};

Quantized quantize(const at::Tensor& x, bool rows, bool columns, int64_t block_rows, at::ScalarType type, bool sums) {
  Quantized r;
  const int64_t m = x.size(0), n = x.size(1);
  zcutlass_quantize_desc d{};
  d.rows = m, d.cols = n, d.ldx = row_stride(x, "x");
  d.x_type = float_code(x, "x"), d.q_type = fp8_code(type, "dtype"), d.block_rows = static_cast<int32_t>(block_rows);
  if (rows) {
    r.q = empty_fp8(m, n, type, x);
    r.scale = block_rows == 1 ? empty_row_scales(m, n, x) : empty_like_device({groups(m), groups(n)}, at::kFloat, x);
    d.ldq = r.q.stride(0), d.scale_row = r.scale.stride(0), d.scale_blk = r.scale.stride(1);
  }
  if (columns) {
    r.qt = empty_fp8(n, m, type, x);
    r.scale_t = block_rows == 1 ? empty_row_scales(n, m, x) : empty_like_device({groups(n), groups(m)}, at::kFloat, x);
    d.ldqt = r.qt.stride(0), d.scale_t_row = r.scale_t.stride(0), d.scale_t_blk = r.scale_t.stride(1);
  }
  if (sums) r.col_sums = empty_like_device({groups(m), n}, at::kFloat, x);
  d.stream = current_stream();
  const auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  check_status(zcutlass_quantize_fp8(&d, x.data_ptr(), ptr(r.q), static_cast<float*>(ptr(r.scale)), ptr(r.qt),
                                     static_cast<float*>(ptr(r.scale_t)), static_cast<float*>(ptr(r.col_sums))),
               "zcutlass_quantize_fp8");
  return r;
}

std::vector<at::Tensor> quantize_fp8_op(const at::Tensor& x, std::string_view layout, std::optional<at::ScalarType> dtype) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a rank-2 CUDA tensor");
  const at::ScalarType t = dtype.value_or(at::kFloat8_e4m3fn);
  const c10::cuda::CUDAGuard guard(x.device());
  if (layout == "rows") {
    const Quantized r = quantize(x, true, false, 1, t, false);
    return {r.q, r.scale};
  }
  if (layout == "columns") {
    const Quantized r = quantize(x, false, true, 1, t, false);
    return {r.qt, r.scale_t};
  }
  if (layout == "both") {
    const Quantized r = quantize(x, true, true, 1, t, false);
    return {r.q, r.scale, r.qt, r.scale_t};
  }
  if (layout == "blocks") {
    const Quantized r = quantize(x, true, false, kFp8Group, t, false);
    return {r.q, r.scale};
  }
  TORCH_CHECK(layout == "blocks_both", "layout must be rows, columns, both, blocks or blocks_both");
  const Quantized r = quantize(x, true, true, kFp8Group, t, false);
  return {r.q, r.scale, r.qt, r.scale_t};
}

void check_fp8_operand(const at::Tensor& t, const at::Tensor& scale, const char* name, bool blocks_allowed) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2, name, " must be a rank-2 CUDA tensor");
  (void)fp8_code(t.scalar_type(), name);
  TORCH_CHECK(scale.is_cuda() && scale.dim() == 2 && scale.scalar_type() == at::kFloat, name,
              "_scale must be a rank-2 float32 CUDA tensor");
  TORCH_CHECK(scale.device() == t.device(), name, "_scale must be on the same CUDA device as ", name);
  const bool per_row = scale.size(0) == t.size(0);
  const bool per_block = blocks_allowed && scale.size(0) == groups(t.size(0));
  TORCH_CHECK((per_row || per_block) && scale.size(1) == groups(t.size(1)), name, "_scale must have shape [",
              blocks_allowed ? "rows or ceil(rows / 128)" : "rows", ", ceil(columns / 128)] of ", name);
}

const void* bias_ptr(const std::optional<at::Tensor>& bias, const at::Tensor& a, at::ScalarType out_type, int64_t n) {
  if (!bias.has_value()) return nullptr;
  TORCH_CHECK(bias->is_cuda() && bias->device() == a.device() && bias->dim() == 1 && bias->is_contiguous(),
              "bias must be a contiguous rank-1 CUDA tensor on the operands' device");
  TORCH_CHECK(bias->scalar_type() == out_type, "bias dtype must match the result's");
  TORCH_CHECK(bias->size(0) == n, "bias length must equal B.shape[0]");
  return bias->data_ptr();
}

at::Tensor run_gemm_fp8(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale,
                        const std::optional<at::Tensor>& bias, at::ScalarType out_type,
                        at::IntArrayRef shape = {}) {
  const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
  at::Tensor d = shape.empty() ? empty_like_device({m, n}, out_type, a) : empty_like_device(shape, out_type, a);
  zcutlass_fp8_gemm_desc g{};
  g.m = m, g.n = n, g.k = k;
  g.lda = row_stride(a, "A"), g.ldb = row_stride(b, "B"), g.ldd = n;
  g.a_type = fp8_code(a.scalar_type(), "A"), g.b_type = fp8_code(b.scalar_type(), "B");
  g.d_type = float_code(d, "out_dtype");
  g.b_scale_rows = b_scale.size(0) == n ? 1 : 128;
  g.a_scale_row = a_scale.stride(0), g.a_scale_blk = a_scale.stride(1);
  g.b_scale_row = b_scale.stride(0), g.b_scale_blk = b_scale.stride(1);
  g.bias = bias_ptr(bias, a, out_type, n);
  g.stream = current_stream();
  check_status(zcutlass_gemm_fp8(&g, a.data_ptr(), a_scale.data_ptr<float>(), b.data_ptr(), b_scale.data_ptr<float>(),
                                 d.data_ptr()),
               "zcutlass_gemm_fp8");
  return d;
}

at::Tensor gemm_fp8_op(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale,
                       const std::optional<at::Tensor>& bias, std::optional<at::ScalarType> out_dtype) {
  check_fp8_operand(a, a_scale, "A", false);
  check_fp8_operand(b, b_scale, "B", true);
  TORCH_CHECK(a.device() == b.device(), "A and B must be on the same CUDA device");
  TORCH_CHECK(a.size(1) == b.size(1), "A.shape[1] must equal B.shape[1]");
  const c10::cuda::CUDAGuard guard(a.device());
  return run_gemm_fp8(a, a_scale, b, b_scale, bias, out_dtype.value_or(at::kBFloat16));
}

// y = x w^T + bias for a matrix x of rows. The quantised x and its scales share one allocation and never
// become tensors: at decode, the calls around two short kernels are most of the time.
at::Tensor run_linear_fp8(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale,
                          const std::optional<at::Tensor>& bias, at::IntArrayRef shape, const at::Tensor& into) {
  const int64_t m = x.size(0), n = w.size(0), k = x.size(1);
  const int64_t ldq = (k + 15) / 16 * 16, q_bytes = m * ldq;
  const at::Tensor buffer = empty_like_device({q_bytes + 4 * m * groups(k)}, at::kByte, x);
  uint8_t* const q = static_cast<uint8_t*>(buffer.data_ptr());
  float* const scale = reinterpret_cast<float*>(q + q_bytes);
  zcutlass_quantize_desc d{};
  d.rows = m, d.cols = k, d.ldx = row_stride(x, "x");
  d.x_type = float_code(x, "x"), d.q_type = ZCUTLASS_E4M3, d.block_rows = 1;
  d.ldq = ldq, d.scale_row = 1, d.scale_blk = m;
  d.stream = current_stream();
  const at::Tensor y = into.defined() ? into : empty_like_device(shape, x.scalar_type(), x);
  zcutlass_fp8_gemm_desc g{};
  g.m = m, g.n = n, g.k = k;
  g.lda = ldq, g.ldb = row_stride(w, "weight"), g.ldd = into.defined() ? row_stride(into, "out") : n;
  g.a_type = ZCUTLASS_E4M3, g.b_type = fp8_code(w.scalar_type(), "weight"), g.d_type = d.x_type;
  g.b_scale_rows = w_scale.size(0) == n ? 1 : 128;
  g.a_scale_row = 1, g.a_scale_blk = m;
  g.b_scale_row = w_scale.stride(0), g.b_scale_blk = w_scale.stride(1);
  g.bias = bias_ptr(bias, x, x.scalar_type(), n);
  g.stream = d.stream;
  check_status(zcutlass_quantize_fp8(&d, x.data_ptr(), q, scale, nullptr, nullptr, nullptr), "zcutlass_quantize_fp8");
  check_status(zcutlass_gemm_fp8(&g, q, scale, w.data_ptr(), w_scale.data_ptr<float>(), y.data_ptr()), "zcutlass_gemm_fp8");
  return y;
}

// x as a matrix [rows, last dimension] of contiguous rows (a copy only where its strides leave no other way).
at::Tensor as_rows(const at::Tensor& x) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  const at::Tensor x2 = x.dim() == 2 ? x : x.reshape({rows, x.size(-1)});
  const bool ok = (x2.size(1) <= 1 || x2.stride(1) == 1) && (rows <= 1 || x2.stride(0) >= x2.size(1));
  return ok ? x2 : x2.contiguous();
}

at::Tensor linear_fp8_op(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale,
                         const std::optional<at::Tensor>& bias) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1, "x must be a CUDA tensor");
  (void)float_code(x, "x");
  check_fp8_operand(w, w_scale, "weight", true);
  TORCH_CHECK(x.device() == w.device(), "x and weight must be on the same CUDA device");
  TORCH_CHECK(x.size(-1) == w.size(1), "x.shape[-1] must equal weight.shape[1]");
  const c10::cuda::CUDAGuard guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = w.size(0);
  return run_linear_fp8(as_rows(x), w, w_scale, bias, shape, at::Tensor());
}

void linear_fp8_out_op(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale,
                       const std::optional<at::Tensor>& bias, at::Tensor out) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a rank-2 CUDA tensor");
  (void)float_code(x, "x");
  check_fp8_operand(w, w_scale, "weight", true);
  TORCH_CHECK(x.device() == w.device() && out.device() == x.device(), "x, weight and out must be on the same CUDA device");
  TORCH_CHECK(x.size(1) == w.size(1), "x.shape[1] must equal weight.shape[1]");
  TORCH_CHECK(out.dim() == 2 && out.size(0) == x.size(0) && out.size(1) == w.size(0),
              "out must be [x.shape[0], weight.shape[0]]");
  TORCH_CHECK(out.scalar_type() == x.scalar_type(), "out dtype must match x");
  const c10::cuda::CUDAGuard guard(x.device());
  run_linear_fp8(as_rows(x), w, w_scale, bias, {}, out);
}

// The differentiable linear keeps x and w in 8 bits, transposed, for its backward pass (undefined where the
// gradient they serve is not wanted).
struct LinearKept {
  at::Tensor y, wt, wt_scale, xt, xt_scale;
};

LinearKept linear_fp8_forward(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, bool need_dx,
                              bool need_dw) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1, "x must be a CUDA tensor");
  TORCH_CHECK(w.is_cuda() && w.dim() == 2, "weight must be a rank-2 CUDA tensor");
  TORCH_CHECK(x.device() == w.device(), "x and weight must be on the same CUDA device");
  TORCH_CHECK(x.size(-1) == w.size(1), "x.shape[-1] must equal weight.shape[1]");
  const c10::cuda::CUDAGuard guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = w.size(0);
  const Quantized qx = quantize(as_rows(x), true, need_dw, 1, at::kFloat8_e4m3fn, false);
  const Quantized qw = quantize(as_rows(w), true, need_dx, kFp8Group, at::kFloat8_e4m3fn, false);
  return {run_gemm_fp8(qx.q, qx.scale, qw.q, qw.scale, bias, x.scalar_type(), shape), qw.qt, qw.scale_t, qx.qt, qx.scale_t};
}

struct LinearGrads {
  at::Tensor dx, dw, db;
};

// dx = Q(dy) Q(w), dw = Q(dy^T) Q(x^T)^T, db = column sums of dy; undefined where not wanted.
LinearGrads linear_fp8_backward(const at::Tensor& grad, const at::Tensor& wt, const at::Tensor& wt_scale, const at::Tensor& xt,
                                const at::Tensor& xt_scale, bool need_dx, bool need_dw, bool need_db, at::ScalarType dw_dtype) {
  LinearGrads g;
  if (!need_dx && !need_dw && !need_db) return g;
  const c10::cuda::CUDAGuard guard(grad.device());
  const at::Tensor dy = as_rows(grad);
  const Quantized r = quantize(dy, need_dx, need_dw || need_db, 1, at::kFloat8_e4m3fn, need_db);
  if (need_dx) {
    std::vector<int64_t> shape(grad.sizes().begin(), grad.sizes().end());
    shape.back() = wt.size(0);
    g.dx = run_gemm_fp8(r.q, r.scale, wt, wt_scale, std::nullopt, dy.scalar_type(), shape);
  }
  if (need_dw) g.dw = run_gemm_fp8(r.qt, r.scale_t, xt, xt_scale, std::nullopt, dw_dtype);
  if (need_db) {
    g.db = empty_like_device({dy.size(1)}, dy.scalar_type(), dy);
    check_status(zcutlass_sum_rows(r.col_sums.data_ptr<float>(), r.col_sums.size(0), dy.size(1), g.db.data_ptr(),
                                   float_code(g.db, "dy"), current_stream()),
                 "zcutlass_sum_rows");
  }
  return g;
}

at::Tensor linear_fp8_train_op(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias) {
  return linear_fp8_forward(x, w, bias, false, false).y;
}

// ---------------------------------------------------------------- rotary positions

constexpr int64_t kMaxHeads = 65536;  // and values of a head: what zcutlass_rotary takes

// The checks of q and k, before anything is allocated or a device is made current.
void check_heads(const at::Tensor& t, const char* name, const at::Tensor& q) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3, name, " must be a rank-3 CUDA tensor [tokens, heads, head_dim]");
  TORCH_CHECK(t.size(1) <= kMaxHeads && t.size(2) <= kMaxHeads, name, " must have at most 65536 heads of at most 65536 values");
  (void)float_code(t, name);
  TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, name, " must have contiguous heads (last dimension)");
  TORCH_CHECK(t.scalar_type() == q.scalar_type() && t.device() == q.device() && t.size(0) == q.size(0) &&
                  t.size(2) == q.size(2),
              "q and k must match in dtype, device, tokens and head_dim");
}

void run_rotary(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_out, const at::Tensor& k_out,
                const at::Tensor& positions, const at::Tensor& table, bool interleaved, bool inverse) {
  TORCH_CHECK(positions.device() == q.device() && table.device() == q.device(),
              "positions and table must be on the device of q and k");
  TORCH_CHECK(positions.dim() == 1 && positions.is_contiguous() && positions.size(0) == q.size(0),
              "positions must be a contiguous rank-1 tensor with one entry per token");
  TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt,
              "positions must be int32 or int64");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kFloat && (table.size(1) <= 1 || table.stride(1) == 1),
              "table must be a float32 matrix [positions, rotary_dim] with contiguous rows");
  TORCH_CHECK(table.size(1) % 2 == 0 && table.size(1) <= q.size(2),
              "table.shape[1] (the rotary dimension) must be even and no more than the head dimension");
  zcutlass_rotary_desc d{};
  d.tokens = q.size(0);
  d.q_heads = static_cast<int32_t>(q.size(1)), d.k_heads = static_cast<int32_t>(k.size(1));
  d.head_dim = static_cast<int32_t>(q.size(2)), d.rotary_dim = static_cast<int32_t>(table.size(1));
  d.dtype = float_code(q, "q"), d.interleaved = interleaved, d.inverse = inverse;
  d.positions64 = positions.scalar_type() == at::kLong;
  d.q_token = q.stride(0), d.q_head = q.stride(1), d.q_out_token = q_out.stride(0), d.q_out_head = q_out.stride(1);
  d.k_token = k.stride(0), d.k_head = k.stride(1), d.k_out_token = k_out.stride(0), d.k_out_head = k_out.stride(1);
  d.table_rows = table.size(0);
  d.table_ld = table.size(0) <= 1 ? table.size(1) : table.stride(0);
  d.stream = current_stream();
  check_status(zcutlass_rotary(&d, q.data_ptr(), q_out.data_ptr(), k.data_ptr(), k_out.data_ptr(), positions.data_ptr(),
                               table.data_ptr<float>()),
               "zcutlass_rotary");
}

std::tuple<at::Tensor, at::Tensor> rotary_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                                             const at::Tensor& table, bool interleaved, bool inverse) {
  check_heads(q, "q", q);
  check_heads(k, "k", q);
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor q_out = empty_like_device(q.sizes(), q.scalar_type(), q), k_out = empty_like_device(k.sizes(), k.scalar_type(), k);
  run_rotary(q, k, q_out, k_out, positions, table, interleaved, inverse);
  return {q_out, k_out};
}

void rotary_inplace_op(at::Tensor q, at::Tensor k, const at::Tensor& positions, const at::Tensor& table,
                       bool interleaved, bool inverse) {
  check_heads(q, "q", q);
  check_heads(k, "k", q);
  at::assert_no_internal_overlap(q);
  at::assert_no_internal_overlap(k);
  at::assert_no_overlap(q, k);
  const c10::cuda::CUDAGuard guard(q.device());
  run_rotary(q, k, q, k, positions, table, interleaved, inverse);
}

// ---------------------------------------------------------------- gradients

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// Forward-mode derivatives: a tensor with a tangent need not require a gradient, and the kernels run below
// autograd, so its tangent would be dropped (in place: kept beside values it no longer belongs to).
template <typename... T>
void check_no_tangent(const char* name, const T&... t) {
  TORCH_CHECK(!((t.defined() && t._fw_grad(0).defined()) || ...), name, " has no forward-mode derivative");
}

// Whether work on `stream` is part of the capture that `id` names (the legacy stream never is).
bool in_capture(const c10::Stream& stream, unsigned long long id) {
  const cudaStream_t s = c10::cuda::CUDAStream(stream).stream();
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long other = 0;
  return s != nullptr && cudaStreamGetCaptureInfo(s, &status, &other) == cudaSuccess &&
         status == cudaStreamCaptureStatusActive && other == id;
}

// While the current stream is being captured: refuses an operand that leads to a leaf whose gradient accumulator
// was made outside the capture and is still alive (an eager graph of the same leaf is). The backward pass would
// wait for that accumulator's stream, which ends the capture, or the process.
void check_capture(const at::Tensor& t) {
  if (!wants_grad(t) || !t.is_cuda()) return;
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(at::cuda::getCurrentCUDAStream(t.get_device()).stream(), &status, &id));
  const auto check = [id](torch::autograd::Node* accumulator) {
    const auto made_on = accumulator->stream();
    TORCH_CHECK(!made_on.has_value() || in_capture(*made_on, id),
                "a graph of this leaf made on another stream is still alive: drop it (its outputs and losses) before "
                "capturing a backward pass");
  };
  if (t.grad_fn() == nullptr) {
    if (const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t)) check(accumulator.get());
    return;
  }
  std::vector<torch::autograd::Node*> left{t.grad_fn().get()};
  std::unordered_set<torch::autograd::Node*> seen(left.begin(), left.end());
  while (!left.empty()) {
    torch::autograd::Node* node = left.back();
    left.pop_back();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node) != nullptr) check(node);
    for (const auto& edge : node->next_edges())
      if (edge.is_valid() && seen.insert(edge.function.get()).second) left.push_back(edge.function.get());
  }
}

template <typename... T>
void check_no_gradient(const char* name, const T&... t) {
  check_no_tangent(name, t...);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(wants_grad(t) || ...), name,
              " has no gradient: use linear_fp8_train, or call it under torch.no_grad()");
}

class LinearFp8 : public torch::autograd::Function<LinearFp8> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const std::optional<at::Tensor>& bias, bool need_dx, bool need_dw, bool need_db) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    const LinearKept kept = linear_fp8_forward(x, w, bias, need_dx, need_dw);
    ctx->save_for_backward({kept.wt, kept.wt_scale, kept.xt, kept.xt_scale});
    ctx->saved_data["w"] = static_cast<int64_t>(w.scalar_type());
    ctx->saved_data["need"] = static_cast<int64_t>((need_dx ? 1 : 0) | (need_dw ? 2 : 0) | (need_db ? 4 : 0));
    return kept.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear_fp8_train has no second derivative (create_graph)");
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const int64_t need = ctx->saved_data["need"].toInt();
    const auto kept = ctx->get_saved_variables();
    // Of the gradients that the operands allow, those that this backward pass asks for.
    LinearGrads g = linear_fp8_backward(grads[0], kept[0], kept[1], kept[2], kept[3],
                                        (need & 1) != 0 && ctx->needs_input_grad(0), (need & 2) != 0 && ctx->needs_input_grad(1),
                                        (need & 4) != 0 && ctx->needs_input_grad(2),
                                        static_cast<at::ScalarType>(ctx->saved_data["w"].toInt()));
    out[0] = std::move(g.dx), out[1] = std::move(g.dw), out[2] = std::move(g.db);
    return out;
  }
};

at::Tensor linear_fp8_train_autograd(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias) {
  const at::Tensor b = bias.value_or(at::Tensor());
  check_no_tangent("linear_fp8_train", x, w, b);
  if (!at::GradMode::is_enabled() || !(wants_grad(x) || wants_grad(w) || wants_grad(b))) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    return linear_fp8_train_op(x, w, bias);
  }
  check_capture(x);
  check_capture(w);
  check_capture(b);
  return LinearFp8::apply(x, w, bias, wants_grad(x), wants_grad(w), wants_grad(b));
}

constexpr char kTableGradient[] = "the table of rotary positions has no gradient: detach it";

class Rotary : public torch::autograd::Function<Rotary> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                               const at::Tensor& table, bool interleaved, bool inverse) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({positions, table});
    ctx->saved_data["mode"] = static_cast<int64_t>((interleaved ? 1 : 0) | (inverse ? 2 : 0));
    auto [qo, ko] = rotary_op(q, k, positions, table, interleaved, inverse);
    return {std::move(qo), std::move(ko)};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

std::tuple<at::Tensor, at::Tensor> rotary_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                                                   const at::Tensor& table, bool interleaved, bool inverse) {
  check_no_tangent("rotary", q, k, table);
  TORCH_CHECK(!at::GradMode::is_enabled() || !wants_grad(table), kTableGradient);
  if (!at::GradMode::is_enabled() || !(wants_grad(q) || wants_grad(k))) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    return rotary_op(q, k, positions, table, interleaved, inverse);
  }
  check_capture(q);
  check_capture(k);
  variable_list out = Rotary::apply(q, k, positions, table, interleaved, inverse);
  return {std::move(out[0]), std::move(out[1])};
}

// The map is linear, its gradient the rotation back: differentiable itself.
variable_list Rotary::backward(AutogradContext* ctx, variable_list grads) {
  const auto kept = ctx->get_saved_variables();
  const int64_t mode = ctx->saved_data["mode"].toInt();
  for (at::Tensor& g : grads)
    if (g.size(2) > 1 && g.stride(2) != 1) g = g.contiguous();
  auto [dq, dk] = rotary_autograd(grads[0], grads[1], kept[0], kept[1], (mode & 1) != 0, (mode & 2) == 0);
  variable_list out(6);
  out[0] = std::move(dq), out[1] = std::move(dk);
  return out;
}

std::vector<at::Tensor> quantize_fp8_autograd(const at::Tensor& x, std::string_view layout, std::optional<at::ScalarType> dtype) {
  check_no_gradient("quantize_fp8", x);
  const at::AutoDispatchBelowADInplaceOrView guard;
  return quantize_fp8_op(x, layout, dtype);
}

at::Tensor gemm_fp8_autograd(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale,
                             const std::optional<at::Tensor>& bias, std::optional<at::ScalarType> out_dtype) {
  check_no_gradient("gemm_fp8", a, b, a_scale, b_scale, bias.value_or(at::Tensor()));
  const at::AutoDispatchBelowADInplaceOrView guard;
  return gemm_fp8_op(a, a_scale, b, b_scale, bias, out_dtype);
}

at::Tensor linear_fp8_autograd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale,
                               const std::optional<at::Tensor>& bias) {
  check_no_gradient("linear_fp8", x, w, w_scale, bias.value_or(at::Tensor()));
  const at::AutoDispatchBelowADInplaceOrView guard;
  return linear_fp8_op(x, w, w_scale, bias);
}

void linear_fp8_out_autograd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale,
                             const std::optional<at::Tensor>& bias, at::Tensor out) {
  check_no_gradient("linear_fp8_out", x, w, w_scale, bias.value_or(at::Tensor()), out);
  const at::AutoDispatchBelowADInplaceOrView guard;
  linear_fp8_out_op(x, w, w_scale, bias, out);
  out.unsafeGetTensorImpl()->bump_version();
}

void rotary_inplace_autograd(at::Tensor q, at::Tensor k, const at::Tensor& positions, const at::Tensor& table,
                             bool interleaved, bool inverse) {
  check_no_tangent("rotary_", q, k, table);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(wants_grad(q) || wants_grad(k)),
              "rotary_ has no gradient: use rotary, or call it under torch.no_grad()");
  TORCH_CHECK(!at::GradMode::is_enabled() || !wants_grad(table), kTableGradient);
  const at::AutoDispatchBelowADInplaceOrView guard;
  rotary_inplace_op(q, k, positions, table, interleaved, inverse);
  // Saved for a backward pass elsewhere, the old values are gone: let autograd see it.
  q.unsafeGetTensorImpl()->bump_version();
  k.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

TORCH_LIBRARY(zcutlass_torch, m) {
  m.def("gemm(Tensor A, Tensor B, Tensor? C=None, Tensor? bias=None, float alpha=1.0, float beta=0.0) -> Tensor");
}

TORCH_LIBRARY_IMPL(zcutlass_torch, CUDA, m) { m.impl("gemm", gemm_op); }

TORCH_LIBRARY(zcutlass, m) {
  m.def("gemm(Tensor A, Tensor B, Tensor? C=None, Tensor? bias=None, float alpha=1.0, float beta=0.0) -> Tensor");
  m.def("gemm_out(Tensor A, Tensor B, Tensor? C, Tensor? bias, float alpha, float beta, Tensor(a!) D) -> ()");
  m.def("linear(Tensor x, Tensor weight, Tensor? bias=None) -> Tensor");
  m.def("quantize_fp8(Tensor x, str layout=\"rows\", ScalarType? dtype=None) -> Tensor[]");
  m.def("gemm_fp8(Tensor A, Tensor A_scale, Tensor B, Tensor B_scale, Tensor? bias=None, ScalarType? out_dtype=None) -> Tensor");
  m.def("linear_fp8(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias=None) -> Tensor");
  m.def("linear_fp8_out(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias, Tensor(a!) out) -> ()");
  m.def("linear_fp8_train(Tensor x, Tensor weight, Tensor? bias=None) -> Tensor");
  m.def("rotary(Tensor q, Tensor k, Tensor positions, Tensor table, bool interleaved=False, bool inverse=False) -> "
        "(Tensor, Tensor)");
  m.def("rotary_(Tensor(a!) q, Tensor(b!) k, Tensor positions, Tensor table, bool interleaved=False, "
        "bool inverse=False) -> ()");
}

TORCH_LIBRARY_IMPL(zcutlass, CUDA, m) {
  m.impl("gemm", gemm_op);
  m.impl("gemm_out", gemm_out_op);
  m.impl("linear", linear_op);
  m.impl("quantize_fp8", quantize_fp8_op);
  m.impl("gemm_fp8", gemm_fp8_op);
  m.impl("linear_fp8", linear_fp8_op);
  m.impl("linear_fp8_out", linear_fp8_out_op);
  m.impl("linear_fp8_train", linear_fp8_train_op);
  m.impl("rotary", rotary_op);
  m.impl("rotary_", rotary_inplace_op);
}

TORCH_LIBRARY_IMPL(zcutlass, Autograd, m) {
  m.impl("quantize_fp8", quantize_fp8_autograd);
  m.impl("gemm_fp8", gemm_fp8_autograd);
  m.impl("linear_fp8", linear_fp8_autograd);
  m.impl("linear_fp8_out", linear_fp8_out_autograd);
  m.impl("linear_fp8_train", linear_fp8_train_autograd);
  m.impl("rotary", rotary_autograd);
  m.impl("rotary_", rotary_inplace_autograd);
}
