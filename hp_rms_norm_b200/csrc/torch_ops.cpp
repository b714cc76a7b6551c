// torch.ops.hp_rms_norm.{rms_norm, relu}: the reference's operator surface,
// implemented on top of the C ABI in include/hp_rms_norm_b200.h.
//
// Mirrors hp_rms_norm/csrc/hp_rms_norm.cpp:4-43 of the reference (the `_C`
// module and the `hp_rms_norm` op namespace with the same op names and
// argument order) and the argument checks of its host wrappers
// (hp_rms_norm/csrc/cuda/hp_rms_norm.cu:12-24, activation_kernels.cu:11-16),
// with the same check messages.  Added on top: dtype/device agreement between
// the tensors, a device guard for the input's device (the reference launches
// on whatever device is current), honest handling of row strides (the
// reference assumes dense rows after view(-1, H)), mutation annotations in the
// schemas and Meta kernels so the ops trace under torch.compile.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <vector>

#include "hp_rms_norm_b200.h"

extern "C" {
// An empty `_C` module: importing it loads this library, whose static
// initialisers register the operators below.
PyObject* PyInit__C(void) {
  static struct PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_C", nullptr, -1, nullptr};
  return PyModule_Create(&module_def);
}
}

namespace {

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return HPRN_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return HPRN_DTYPE_FP16;
  TORCH_CHECK(false, "dtype must be kFloat16 or kBFloat16");
}

// Rows of a [..., hidden] tensor whose last dim is contiguous: the number of
// rows and the stride between consecutive rows, or an error when the leading
// dims cannot be walked with one stride (the case where the reference's
// view(-1, hidden) throws).
void rows_of(const at::Tensor& t, const char* name, int64_t* rows, int64_t* stride) {
  const int64_t hidden = t.size(-1);
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  *rows = n;
  *stride = hidden;
  if (n <= 1) return;
  int64_t expect = -1;  // stride the next-outer non-trivial dim must have
  int64_t row_stride = -1;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (row_stride < 0) {
      row_stride = t.stride(i);
      expect = t.stride(i) * t.size(i);
    } else {
      TORCH_CHECK(t.stride(i) == expect, name,
                  " must be viewable as (-1, hidden_dim): its leading dimensions are not "
                  "collapsible into rows of one stride");
      expect = t.stride(i) * t.size(i);
    }
  }
  *stride = row_stride;
}

void check_status(int status) {
  TORCH_CHECK(status == HPRN_OK, hprn_status_string(status), ": ", hprn_last_error());
}

void rms_norm(at::Tensor& input, const at::Tensor& weight, at::Tensor& residual, double eps) {
  // hp_rms_norm/csrc/cuda/hp_rms_norm.cu:12-24
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(input.dim() == residual.dim(), "input.dim() == residual.dim()");
  for (int64_t i = 0; i < input.dim(); ++i) {
    TORCH_CHECK(input.size(i) == residual.size(i), "input.size(i) == residual.size(i)");
  }
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  const int64_t hidden = weight.size(0);
  TORCH_CHECK(input.size(-1) == hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(input.stride(-1) == 1, "input.stride(-1) == 1");
  TORCH_CHECK(residual.stride(-1) == 1, "residual.stride(-1) == 1");
  // Added checks.
  TORCH_CHECK(input.is_cuda() && weight.is_cuda() && residual.is_cuda(),
              "input, weight and residual must be CUDA tensors");
  TORCH_CHECK(weight.device() == input.device() && residual.device() == input.device(),
              "input, weight and residual must be on the same device");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type() &&
                  residual.scalar_type() == input.scalar_type(),
              "input, weight and residual must have the same dtype");
  TORCH_CHECK(hidden <= 1 || weight.stride(0) == 1, "weight must be contiguous");
  const int dtype = dtype_code(input);
  int64_t rows = 0, xs = 0, rrows = 0, rs = 0;
  rows_of(input, "input", &rows, &xs);
  rows_of(residual, "residual", &rrows, &rs);
  if (rows == 0 || hidden == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_rms_norm(input.data_ptr(), weight.data_ptr(), residual.data_ptr(), rows, hidden,
                             xs, rs, eps, dtype, stream));
}

void relu(at::Tensor& out, const at::Tensor& input) {
  // hp_rms_norm/csrc/cuda/activation_kernels.cu:11-16
  TORCH_CHECK(input.dim() >= 2, "input.dim() >= 2");
  TORCH_CHECK(input.dim() == out.dim(), "input.size(i) == out.size(i)");
  for (int64_t i = 0; i < input.dim(); ++i) {
    TORCH_CHECK(input.size(i) == out.size(i), "input.size(i) == out.size(i)");
  }
  // Added checks.
  TORCH_CHECK(input.is_cuda() && out.is_cuda(), "out and input must be CUDA tensors");
  TORCH_CHECK(out.device() == input.device(), "out and input must be on the same device");
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), "out and input must have the same dtype");
  const int dtype = dtype_code(input);
  const int64_t hidden = input.size(-1);
  if (input.numel() == 0) return;
  TORCH_CHECK(hidden == 1 || input.stride(-1) == 1, "input.stride(-1) == 1");
  TORCH_CHECK(hidden == 1 || out.stride(-1) == 1, "out.stride(-1) == 1");
  int64_t rows = 0, is = 0, orows = 0, os = 0;
  rows_of(input, "input", &rows, &is);
  rows_of(out, "out", &orows, &os);
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_relu(out.data_ptr(), input.data_ptr(), rows, hidden, os, is, dtype, stream));
}

// Common checks of the out-of-place forms (extensions past the reference).
struct OutCall {
  int64_t rows = 0, hidden = 0, os = 0, xs = 0, rs = 0;
  int dtype = 0;
};

OutCall check_out_call(const at::Tensor& out, const at::Tensor& input, const at::Tensor& weight,
                       const c10::optional<at::Tensor>& residual) {
  OutCall c;
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  c.hidden = weight.size(0);
  TORCH_CHECK(input.size(-1) == c.hidden, "input.size(-1) == hidden_dim");
  TORCH_CHECK(out.sizes() == input.sizes(), "out must have the input's shape");
  TORCH_CHECK(input.is_cuda() && weight.is_cuda() && out.is_cuda(), "tensors must be CUDA tensors");
  TORCH_CHECK(weight.device() == input.device() && out.device() == input.device(),
              "tensors must be on the same device");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), "input and weight must have the same dtype");
  TORCH_CHECK(c.hidden <= 1 || weight.stride(0) == 1, "weight must be contiguous");
  TORCH_CHECK(input.stride(-1) == 1 || c.hidden == 1, "input.stride(-1) == 1");
  TORCH_CHECK(out.stride(-1) == 1 || c.hidden == 1, "out.stride(-1) == 1");
  c.dtype = dtype_code(input);
  rows_of(input, "input", &c.rows, &c.xs);
  int64_t orows = 0;
  rows_of(out, "out", &orows, &c.os);
  c.rs = c.hidden;
  if (residual.has_value()) {
    const at::Tensor& r = *residual;
    TORCH_CHECK(r.sizes() == input.sizes(), "residual must have the input's shape");
    TORCH_CHECK(r.is_cuda() && r.device() == input.device(), "residual must be on the input's device");
    TORCH_CHECK(r.scalar_type() == input.scalar_type(), "input and residual must have the same dtype");
    TORCH_CHECK(r.stride(-1) == 1 || c.hidden == 1, "residual.stride(-1) == 1");
    int64_t rrows = 0;
    rows_of(r, "residual", &rrows, &c.rs);
  }
  return c;
}

// out <- RMSNorm(input [+ residual]) * weight in the input's dtype; the
// residual (if given) is updated in place; out may be the input itself.
void rms_norm_out(at::Tensor& out, const at::Tensor& input, const at::Tensor& weight,
                  c10::optional<at::Tensor> residual, double eps) {
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), "out must have the input's dtype");
  const OutCall c = check_out_call(out, input, weight, residual);
  if (c.rows == 0 || c.hidden == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_rms_norm_out(out.data_ptr(), input.data_ptr(), weight.data_ptr(),
                                 residual.has_value() ? residual->data_ptr() : nullptr, c.rows,
                                 c.hidden, c.os, c.xs, c.rs, eps, c.dtype, HPRN_OUT_SAME, nullptr,
                                 nullptr, stream, HPRN_LAUNCH_DEFAULT));
}

// out (float8_e4m3fn) <- e4m3(RMSNorm(input [+ residual]) * weight / scale):
// with `scale` (one float32) a static per-tensor scale, with `row_scales`
// (float32 [rows], written) a per-row scale max|y| / 448.
void rms_norm_fp8(at::Tensor& out, const at::Tensor& input, const at::Tensor& weight,
                  c10::optional<at::Tensor> residual, double eps, c10::optional<at::Tensor> scale,
                  c10::optional<at::Tensor> row_scales) {
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "out must be float8_e4m3fn");
  TORCH_CHECK(scale.has_value() != row_scales.has_value(),
              "exactly one of scale (static) and row_scales (dynamic) must be given");
  const OutCall c = check_out_call(out, input, weight, residual);
  const float* sp = nullptr;
  float* rsp = nullptr;
  if (scale.has_value()) {
    TORCH_CHECK(scale->scalar_type() == at::kFloat && scale->numel() == 1 && scale->is_cuda() &&
                    scale->device() == input.device(),
                "scale must be one float32 on the input's device");
    sp = scale->data_ptr<float>();
  } else {
    TORCH_CHECK(row_scales->scalar_type() == at::kFloat && row_scales->numel() == c.rows &&
                    row_scales->is_contiguous() && row_scales->is_cuda() &&
                    row_scales->device() == input.device(),
                "row_scales must be a contiguous float32 tensor with one entry per row");
    rsp = row_scales->data_ptr<float>();
  }
  if (c.rows == 0 || c.hidden == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_rms_norm_out(out.data_ptr(), input.data_ptr(), weight.data_ptr(),
                                 residual.has_value() ? residual->data_ptr() : nullptr, c.rows,
                                 c.hidden, c.os, c.xs, c.rs, eps, c.dtype,
                                 sp ? HPRN_OUT_FP8_E4M3_STATIC : HPRN_OUT_FP8_E4M3_DYNAMIC, sp,
                                 rsp, stream, HPRN_LAUNCH_DEFAULT));
}

// NVFP4 output (extension past the reference): out uint8 [..., hidden/2] holds
// e2m1 pairs (element 2k in the low nibble), block_scales (uint8 or
// float8_e4m3fn) [..., hidden/16] one e4m3 scale per 16 elements, global_scale
// one float32: y ~ e2m1 * scale / global_scale.
void rms_norm_nvfp4(at::Tensor& out, at::Tensor& block_scales, const at::Tensor& input,
                    const at::Tensor& weight, c10::optional<at::Tensor> residual, double eps,
                    const at::Tensor& global_scale) {
  TORCH_CHECK(input.dim() >= 1 && weight.dim() == 1 && input.size(-1) == weight.size(0),
              "input.size(-1) == hidden_dim");
  const int64_t hidden = weight.size(0);
  TORCH_CHECK(hidden % 16 == 0, "NVFP4 output needs hidden_dim % 16 == 0");
  TORCH_CHECK(out.scalar_type() == at::kByte, "out must be uint8 (two e2m1 codes per byte)");
  TORCH_CHECK(block_scales.scalar_type() == at::kByte ||
                  block_scales.scalar_type() == at::kFloat8_e4m3fn,
              "block_scales must be uint8 or float8_e4m3fn");
  TORCH_CHECK(out.dim() == input.dim() && block_scales.dim() == input.dim(),
              "out and block_scales must have the input's rank");
  for (int64_t i = 0; i + 1 < input.dim(); ++i)
    TORCH_CHECK(out.size(i) == input.size(i) && block_scales.size(i) == input.size(i),
                "out and block_scales must agree with the input on leading dimensions");
  TORCH_CHECK(out.size(-1) == hidden / 2 && block_scales.size(-1) == hidden / 16,
              "out.size(-1) == hidden_dim / 2 and block_scales.size(-1) == hidden_dim / 16");
  TORCH_CHECK(block_scales.is_contiguous(), "block_scales must be contiguous");
  TORCH_CHECK(global_scale.scalar_type() == at::kFloat && global_scale.numel() == 1,
              "global_scale must be one float32");
  const at::Tensor* all[] = {&out, &block_scales, &input, &weight, &global_scale};
  for (const at::Tensor* t : all)
    TORCH_CHECK(t->is_cuda() && t->device() == input.device(), "tensors must share a CUDA device");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), "input and weight must have the same dtype");
  TORCH_CHECK(input.stride(-1) == 1 && out.stride(-1) == 1 && weight.stride(0) == 1,
              "input, out and weight must be contiguous in the last dimension");
  const int dtype = dtype_code(input);
  int64_t rows = 0, xs = 0, orows = 0, os = 0, rs = hidden;
  rows_of(input, "input", &rows, &xs);
  rows_of(out, "out", &orows, &os);
  void* rp = nullptr;
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == input.sizes() && residual->scalar_type() == input.scalar_type() &&
                    residual->is_cuda() && residual->device() == input.device() &&
                    residual->stride(-1) == 1,
                "residual must match the input's shape, dtype and device");
    int64_t rrows = 0;
    rows_of(*residual, "residual", &rrows, &rs);
    rp = residual->data_ptr();
  }
  if (rows == 0 || hidden == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_rms_norm_nvfp4(out.data_ptr(), static_cast<uint8_t*>(block_scales.data_ptr()),
                                   input.data_ptr(), weight.data_ptr(), rp, rows, hidden, os * 2,
                                   xs, rs, eps, dtype, global_scale.data_ptr<float>(), stream,
                                   HPRN_LAUNCH_DEFAULT));
}

// Per-token-group fp8 output (extension past the reference): out
// float8_e4m3fn [..., hidden]; scales float32 [rows, hidden / group_size]
// (rows = the input's leading dimensions flattened), any strides, so a
// transposed view gives column-major scales.
void rms_norm_fp8_group(at::Tensor& out, at::Tensor& scales, const at::Tensor& input,
                        const at::Tensor& weight, c10::optional<at::Tensor> residual, double eps,
                        int64_t group_size, bool scale_pow2) {
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "out must be float8_e4m3fn");
  const OutCall c = check_out_call(out, input, weight, residual);
  TORCH_CHECK(group_size == 32 || group_size == 64 || group_size == 128,
              "group_size must be 32, 64 or 128");
  TORCH_CHECK(c.hidden % group_size == 0, "hidden_dim must be a multiple of group_size");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.dim() == 2 &&
                  scales.size(0) == c.rows && scales.size(1) == c.hidden / group_size,
              "scales must be float32 [rows, hidden / group_size]");
  TORCH_CHECK(scales.is_cuda() && scales.device() == input.device(),
              "scales must be on the input's device");
  if (c.rows == 0 || c.hidden == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_rms_norm_fp8_group(
      out.data_ptr(), scales.data_ptr<float>(), scales.stride(0), scales.stride(1),
      input.data_ptr(), weight.data_ptr(), residual.has_value() ? residual->data_ptr() : nullptr,
      c.rows, c.hidden, c.os, c.xs, c.rs, eps, c.dtype, static_cast<int>(group_size),
      scale_pow2 ? 1 : 0, stream, HPRN_LAUNCH_DEFAULT));
}

// out[..., d] = act(input[..., :d]) * input[..., d:]  (extension past the reference).
void act_and_mul(at::Tensor& out, const at::Tensor& input, int act) {
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) % 2 == 0, "input.size(-1) must be even");
  const int64_t d = input.size(-1) / 2;
  TORCH_CHECK(out.dim() == input.dim(), "out.dim() == input.dim()");
  for (int64_t i = 0; i + 1 < input.dim(); ++i)
    TORCH_CHECK(out.size(i) == input.size(i), "out and input must agree on leading dimensions");
  TORCH_CHECK(out.size(-1) == d, "out.size(-1) == input.size(-1) / 2");
  TORCH_CHECK(input.is_cuda() && out.is_cuda() && out.device() == input.device(),
              "out and input must be CUDA tensors on the same device");
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), "out and input must have the same dtype");
  const int dtype = dtype_code(input);
  if (out.numel() == 0) return;
  TORCH_CHECK(input.stride(-1) == 1 && (d == 1 || out.stride(-1) == 1),
              "input and out must be contiguous in the last dimension");
  int64_t rows = 0, is = 0, orows = 0, os = 0;
  rows_of(input, "input", &rows, &is);
  rows_of(out, "out", &orows, &os);
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_act_and_mul(out.data_ptr(), input.data_ptr(), rows, d, os, is, act, dtype,
                                stream, HPRN_LAUNCH_DEFAULT));
}

void silu_and_mul(at::Tensor& out, const at::Tensor& input) { act_and_mul(out, input, HPRN_ACT_SILU); }
void gelu_and_mul(at::Tensor& out, const at::Tensor& input) { act_and_mul(out, input, HPRN_ACT_GELU); }
void gelu_tanh_and_mul(at::Tensor& out, const at::Tensor& input) {
  act_and_mul(out, input, HPRN_ACT_GELU_TANH);
}

// ---------------------------------------------------------------------------
// Training operators (extensions past the reference).

// A [..., cols] tensor as rows of one stride on `like`'s device.
struct Rows {
  void* p = nullptr;
  int64_t rows = 0, stride = 0;
};

Rows rows_arg(const at::Tensor& t, const char* name, int64_t cols, const at::Tensor& like,
              at::ScalarType type) {
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) == cols, name, ".size(-1) must be ", cols);
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name,
              " must be a CUDA tensor on the same device as the others");
  TORCH_CHECK(t.scalar_type() == type, name, " must be of dtype ", type);
  TORCH_CHECK(cols <= 1 || t.numel() == 0 || t.stride(-1) == 1, name, ".stride(-1) == 1");
  Rows r;
  if (t.numel() > 0 || cols == 0) {
    rows_of(t, name, &r.rows, &r.stride);
  } else {
    r.rows = 0, r.stride = cols;
  }
  if (r.rows <= 1) r.stride = cols;  // never stepped over
  r.p = t.data_ptr();
  return r;
}

// Same rows as `like` (the leading dimensions, not just their product).
void check_leading(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.dim() == like.dim(), name, " must have as many dimensions as input");
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    TORCH_CHECK(t.size(i) == like.size(i), name, " and input must agree on leading dimensions");
}

const float* float_rows(const at::Tensor& t, const char* name, int64_t rows, const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == rows && t.is_contiguous() &&
                  t.is_cuda() && t.device() == like.device(),
              name, " must be a contiguous float32 tensor with one entry per row");
  return t.data_ptr<float>();
}

const int64_t* target_rows(const at::Tensor& t, int64_t rows, const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kLong && t.numel() == rows && t.is_contiguous() &&
                  t.is_cuda() && t.device() == like.device(),
              "target must be a contiguous int64 tensor with one entry per row");
  return t.data_ptr<int64_t>();
}

// Device memory of one call, from torch's caching allocator without a tensor
// around it (1 us less a call).  Given back at once: the allocator hands it on
// to later work of the same stream only.
class StreamMemory {
 public:
  StreamMemory(int64_t bytes, cudaStream_t stream) {
    if (bytes > 0)
      p_ = c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(static_cast<size_t>(bytes), stream);
  }
  ~StreamMemory() {
    if (p_) c10::cuda::CUDACachingAllocator::raw_delete(p_);
  }
  StreamMemory(const StreamMemory&) = delete;
  StreamMemory& operator=(const StreamMemory&) = delete;
  void* get() const { return p_; }

 private:
  void* p_ = nullptr;
};

// Runs an entry point twice: once for the size of its workspace, once with one.
template <typename F>
void with_workspace(const at::Tensor& like, F&& call) {
  const c10::cuda::CUDAGuard guard(like.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(like.device().index()).stream();
  int64_t bytes = 0;
  check_status(call(nullptr, &bytes, stream, HPRN_WORKSPACE_QUERY));
  const StreamMemory ws(bytes, stream);
  check_status(call(ws.get(), &bytes, stream, HPRN_LAUNCH_DEFAULT));
}

int act_code(c10::string_view act) {
  if (act == "silu") return HPRN_ACT_SILU;
  if (act == "gelu") return HPRN_ACT_GELU;
  if (act == "gelu_tanh") return HPRN_ACT_GELU_TANH;
  TORCH_CHECK(false, "act must be 'silu', 'gelu' or 'gelu_tanh'");
}

struct GatedCall {
  int act, dtype;
  int64_t hidden, d;
  Rows x, w;
};

GatedCall check_gated(const at::Tensor& input, const at::Tensor& weight, c10::string_view act) {
  GatedCall c;
  c.act = act_code(act);
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) % 2 == 0, "weight must be [2 * d, hidden]");
  c.dtype = dtype_code(input);
  c.hidden = input.size(-1);
  c.d = weight.size(0) / 2;
  c.x = rows_arg(input, "input", c.hidden, input, input.scalar_type());
  c.w = rows_arg(weight, "weight", c.hidden, input, input.scalar_type());
  return c;
}

// rows of a [..., cols] tensor, its last dimension included when that is 0.
int64_t leading(const at::Tensor& t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  return n;
}

void gated_linear(at::Tensor& out, c10::optional<at::Tensor> gate_up, const at::Tensor& input,
                  const at::Tensor& weight, c10::string_view act) {
  const GatedCall c = check_gated(input, weight, act);
  const int64_t rows = leading(input);
  check_leading(out, "out", input);
  const Rows o = rows_arg(out, "out", c.d, input, input.scalar_type());
  Rows g;
  if (gate_up.has_value()) {
    check_leading(*gate_up, "gate_up", input);
    g = rows_arg(*gate_up, "gate_up", 2 * c.d, input, at::kFloat);
  }
  if (rows == 0 || c.d == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_gated_linear(o.p, static_cast<float*>(g.p), c.x.p, c.w.p, rows, c.hidden, c.d,
                             o.stride, g.stride, c.x.stride, c.w.stride, c.act, c.dtype, ws, bytes,
                             s, flags);
  });
}

void gated_linear_backward(at::Tensor& grad_input, at::Tensor& grad_weight,
                           const at::Tensor& grad_out, const at::Tensor& input,
                           const at::Tensor& weight, c10::optional<at::Tensor> gate_up,
                           c10::string_view act) {
  const GatedCall c = check_gated(input, weight, act);
  const int64_t rows = leading(input);
  check_leading(grad_out, "grad_out", input);
  check_leading(grad_input, "grad_input", input);
  TORCH_CHECK(grad_weight.sizes() == weight.sizes(), "grad_weight must have the weight's shape");
  const Rows d = rows_arg(grad_out, "grad_out", c.d, input, input.scalar_type());
  const Rows gi = rows_arg(grad_input, "grad_input", c.hidden, input, input.scalar_type());
  const Rows gw = rows_arg(grad_weight, "grad_weight", c.hidden, input, input.scalar_type());
  Rows g;
  if (gate_up.has_value()) {
    check_leading(*gate_up, "gate_up", input);
    g = rows_arg(*gate_up, "gate_up", 2 * c.d, input, at::kFloat);
  }
  if (c.hidden == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_gated_linear_backward(gi.p, gw.p, d.p, static_cast<const float*>(g.p), c.x.p, c.w.p,
                                      rows, c.hidden, c.d, gi.stride, gw.stride, d.stride, g.stride,
                                      c.x.stride, c.w.stride, c.act, c.dtype, ws, bytes, s, flags);
  });
}

struct LossCall {
  int dtype;
  int64_t rows, hidden, vocab;
  Rows x, w;
  const int64_t* target;
};

LossCall check_loss(const at::Tensor& input, const at::Tensor& weight, const at::Tensor& target) {
  LossCall c;
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 2, "weight must be [vocab, hidden]");
  c.dtype = dtype_code(input);
  c.rows = leading(input);
  c.hidden = input.size(-1);
  c.vocab = weight.size(0);
  c.x = rows_arg(input, "input", c.hidden, input, input.scalar_type());
  c.w = rows_arg(weight, "weight", c.hidden, input, input.scalar_type());
  c.target = target_rows(target, c.rows, input);
  return c;
}

void linear_cross_entropy(at::Tensor& loss, at::Tensor& lse, const at::Tensor& input,
                          const at::Tensor& weight, const at::Tensor& target, int64_t ignore_index) {
  const LossCall c = check_loss(input, weight, target);
  float* lp = const_cast<float*>(float_rows(loss, "loss", c.rows, input));
  float* ep = const_cast<float*>(float_rows(lse, "lse", c.rows, input));
  if (c.rows == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_linear_cross_entropy(lp, ep, c.x.p, c.w.p, c.target, ignore_index, c.rows, c.hidden,
                                     c.vocab, c.x.stride, c.w.stride, c.dtype, ws, bytes, s, flags);
  });
}

void linear_cross_entropy_backward(at::Tensor& grad_input, at::Tensor& grad_weight,
                                   const at::Tensor& grad_loss, const at::Tensor& input,
                                   const at::Tensor& weight, const at::Tensor& target,
                                   const at::Tensor& lse, int64_t ignore_index) {
  const LossCall c = check_loss(input, weight, target);
  TORCH_CHECK(grad_input.sizes() == input.sizes(), "grad_input must have the input's shape");
  TORCH_CHECK(grad_weight.sizes() == weight.sizes(), "grad_weight must have the weight's shape");
  const Rows gi = rows_arg(grad_input, "grad_input", c.hidden, input, input.scalar_type());
  const Rows gw = rows_arg(grad_weight, "grad_weight", c.hidden, input, input.scalar_type());
  const float* gl = float_rows(grad_loss, "grad_loss", c.rows, input);
  const float* ep = float_rows(lse, "lse", c.rows, input);
  if (c.hidden == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_linear_cross_entropy_backward(gi.p, gw.p, gl, c.x.p, c.w.p, c.target, ep,
                                              ignore_index, c.rows, c.hidden, c.vocab, gi.stride,
                                              gw.stride, c.x.stride, c.w.stride, c.dtype, ws, bytes,
                                              s, flags);
  });
}

void rms_norm_backward(at::Tensor& grad_input, at::Tensor& grad_weight, const at::Tensor& grad_out,
                       const at::Tensor& input, const at::Tensor& weight,
                       c10::optional<at::Tensor> grad_residual, double eps) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  const int64_t hidden = weight.size(0);
  TORCH_CHECK(input.size(-1) == hidden, "input.size(-1) == hidden_dim");
  const int dtype = dtype_code(input);
  const at::ScalarType type = input.scalar_type();
  const int64_t rows = leading(input);
  TORCH_CHECK(grad_out.sizes() == input.sizes(), "grad_out must have the input's shape");
  TORCH_CHECK(grad_input.sizes() == input.sizes(), "grad_input must have the input's shape");
  TORCH_CHECK(grad_weight.dim() == 1, "grad_weight.dim() == 1");
  const Rows x = rows_arg(input, "input", hidden, input, type);
  const Rows w = rows_arg(weight, "weight", hidden, input, type);
  const Rows d = rows_arg(grad_out, "grad_out", hidden, input, type);
  const Rows gi = rows_arg(grad_input, "grad_input", hidden, input, type);
  const Rows gw = rows_arg(grad_weight, "grad_weight", hidden, input, type);
  Rows r;
  if (grad_residual.has_value()) {
    TORCH_CHECK(grad_residual->sizes() == input.sizes(), "grad_residual must have the input's shape");
    r = rows_arg(*grad_residual, "grad_residual", hidden, input, type);
  }
  if (hidden == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_rms_norm_backward(gi.p, gw.p, d.p, x.p, w.p, r.p, rows, hidden, gi.stride, d.stride,
                                  x.stride, r.stride, eps, dtype, ws, bytes, s, flags);
  });
}

int32_t grad_dtype(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return HPRN_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return HPRN_DTYPE_FP16;
  if (t.scalar_type() == at::kFloat) return HPRN_DTYPE_FP32;
  TORCH_CHECK(false, "gradients must be kFloat16, kBFloat16 or kFloat");
}

// rows, cols and row stride of a tensor whose elements are taken in order.
void grad_layout(const at::Tensor& t, const char* name, int64_t* rows, int64_t* cols, int64_t* stride) {
  if (t.is_contiguous()) {
    *rows = 1, *cols = t.numel(), *stride = t.numel();
    return;
  }
  *cols = t.size(-1);
  TORCH_CHECK(t.size(-1) == 1 || t.stride(-1) == 1, name,
              " must be contiguous in its last dimension");
  rows_of(t, name, rows, stride);
}

std::vector<hprn_grad> grad_table(at::TensorList grads, const at::TensorList* outs,
                                  const at::Tensor& norm) {
  TORCH_CHECK(norm.is_cuda() && norm.scalar_type() == at::kFloat && norm.numel() == 1,
              "norm must be one float32 on the gradients' device");
  std::vector<hprn_grad> table(grads.size());
  for (size_t k = 0; k < grads.size(); ++k) {
    const at::Tensor& t = grads[k];
    hprn_grad& e = table[k];
    TORCH_CHECK(t.is_cuda() && t.device() == norm.device(),
                "gradients must be CUDA tensors on one device");
    e.dtype = e.out_dtype = grad_dtype(t);
    grad_layout(t, "gradients", &e.rows, &e.cols, &e.row_stride);
    e.grad = t.data_ptr(), e.out = nullptr, e.out_row_stride = e.row_stride;
    if (!outs) continue;
    const at::Tensor& o = (*outs)[k];
    TORCH_CHECK(o.is_cuda() && o.device() == norm.device(), "out must be on the gradients' device");
    TORCH_CHECK(o.sizes() == t.sizes(), "out must have the gradients' shapes");
    e.out_dtype = grad_dtype(o);
    e.out = o.data_ptr();
    int64_t orows = 0, ocols = 0;
    grad_layout(o, "out", &orows, &ocols, &e.out_row_stride);
    if (orows == e.rows && ocols == e.cols) continue;
    // One of the two is contiguous, the other has rows: walk both by its rows.
    if (e.rows == 1) {
      e.rows = orows, e.cols = ocols, e.row_stride = ocols;
    } else if (orows == 1) {
      e.out_row_stride = e.cols;
    }
  }
  return table;
}

void grad_norm(at::Tensor& norm, at::TensorList grads) {
  const std::vector<hprn_grad> table = grad_table(grads, nullptr, norm);
  with_workspace(norm, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_grad_norm(norm.data_ptr<float>(), table.data(), static_cast<int64_t>(table.size()), ws,
                          bytes, s, flags);
  });
}

void clip_grad_norm(at::TensorList out, at::Tensor& norm, at::TensorList grads, double max_norm) {
  TORCH_CHECK(out.size() == grads.size(), "out must have one tensor per gradient");
  const std::vector<hprn_grad> table = grad_table(grads, &out, norm);
  with_workspace(norm, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_clip_grad_norm(norm.data_ptr<float>(), table.data(), static_cast<int64_t>(table.size()),
                               max_norm, ws, bytes, s, flags);
  });
}

// A gate over `input`: rows of `width` (1 or hidden) values, each for the rows of
// input that the gate's trailing dimensions of 1 span.
struct Gate {
  Rows rows;
  int64_t width = 1, rows_per_gate = 1;
};

Gate gate_arg(const at::Tensor& gate, const char* name, const at::Tensor& input) {
  TORCH_CHECK(gate.dim() >= 1 && gate.dim() <= input.dim(), name, " must have 1 to input.dim() dimensions");
  Gate g;
  g.width = gate.size(-1);
  TORCH_CHECK(g.width == input.size(-1) || g.width == 1, name, ".size(-1) must be 1 or hidden_dim");
  // From the last leading dimension outwards: dimensions of 1, then input's own.
  bool own = false;
  for (int64_t k = 2; k <= input.dim(); ++k) {
    const int64_t n = k <= gate.dim() ? gate.size(-k) : 1, of = input.size(-k);
    TORCH_CHECK(n == of || (n == 1 && !own), name,
                " must broadcast over input's trailing leading dimensions only");
    if (n != of) g.rows_per_gate *= of;
    own = own || (n == of && n != 1);
  }
  g.rows = rows_arg(gate, name, g.width, input, input.scalar_type());
  return g;
}

struct BlockNorm {
  int dtype;
  int64_t hidden, rows, rows_per_gate = 1, gate_width = 1;
  Rows x, p, w, g;
};

BlockNorm check_block_norm(const at::Tensor& input, const c10::optional<at::Tensor>& post_weight,
                           const at::Tensor& weight, const c10::optional<at::Tensor>& gate) {
  BlockNorm c;
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 1, "weight.dim() == 1");
  c.hidden = weight.size(0);
  TORCH_CHECK(input.size(-1) == c.hidden, "input.size(-1) == hidden_dim");
  c.dtype = dtype_code(input);
  c.rows = leading(input);
  c.x = rows_arg(input, "input", c.hidden, input, input.scalar_type());
  c.w = rows_arg(weight, "weight", c.hidden, input, input.scalar_type());
  if (post_weight.has_value()) {
    TORCH_CHECK(post_weight->dim() == 1, "post_weight.dim() == 1");
    c.p = rows_arg(*post_weight, "post_weight", c.hidden, input, input.scalar_type());
  }
  if (gate.has_value()) {
    const Gate g = gate_arg(*gate, "gate", input);
    c.g = g.rows, c.gate_width = g.width, c.rows_per_gate = g.rows_per_gate > 0 ? g.rows_per_gate : 1;
  }
  return c;
}

// The new residual in a tensor of its own.
void gated_add_rms_norm_sum(at::Tensor& out, at::Tensor& total, const at::Tensor& input,
                            const at::Tensor& residual, c10::optional<at::Tensor> post_weight,
                            const at::Tensor& weight, c10::optional<at::Tensor> gate,
                            double residual_scale, double eps) {
  const BlockNorm c = check_block_norm(input, post_weight, weight, gate);
  const at::ScalarType type = input.scalar_type();
  TORCH_CHECK(out.sizes() == input.sizes(), "out must have the input's shape");
  TORCH_CHECK(residual.sizes() == input.sizes(), "residual must have the input's shape");
  TORCH_CHECK(total.sizes() == input.sizes(), "residual_out must have the input's shape");
  const Rows o = rows_arg(out, "out", c.hidden, input, type);
  const Rows r = rows_arg(residual, "residual", c.hidden, input, type);
  const Rows t = rows_arg(total, "residual_out", c.hidden, input, type);
  if (c.rows == 0 || c.hidden == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_gated_add_rms_norm(o.p, t.p, c.x.p, r.p, c.p.p, c.w.p, c.g.p, c.rows, c.hidden,
                                       c.rows_per_gate, c.gate_width, o.stride, t.stride, c.x.stride,
                                       r.stride, c.g.stride, residual_scale, eps, c.dtype, stream,
                                       HPRN_LAUNCH_DEFAULT));
}

void gated_add_rms_norm(at::Tensor& out, at::Tensor& residual, c10::optional<at::Tensor> residual_out,
                        const at::Tensor& input, c10::optional<at::Tensor> post_weight,
                        const at::Tensor& weight, c10::optional<at::Tensor> gate,
                        double residual_scale, double eps) {
  gated_add_rms_norm_sum(out, residual_out.has_value() ? *residual_out : residual, input, residual, post_weight,
                         weight, gate, residual_scale, eps);
}

void gated_add_rms_norm_backward(at::Tensor& grad_input, at::Tensor& grad_residual,
                                 c10::optional<at::Tensor> grad_post_weight, at::Tensor& grad_weight,
                                 c10::optional<at::Tensor> grad_gate, const at::Tensor& grad_out,
                                 c10::optional<at::Tensor> grad_residual_out,
                                 const at::Tensor& input, const at::Tensor& residual_out,
                                 c10::optional<at::Tensor> post_weight, const at::Tensor& weight,
                                 c10::optional<at::Tensor> gate, double residual_scale, double eps) {
  const BlockNorm c = check_block_norm(input, post_weight, weight, gate);
  const at::ScalarType type = input.scalar_type();
  TORCH_CHECK(grad_out.sizes() == input.sizes(), "grad_out must have the input's shape");
  TORCH_CHECK(residual_out.sizes() == input.sizes(), "residual must have the input's shape");
  TORCH_CHECK(grad_input.sizes() == input.sizes(), "grad_input must have the input's shape");
  TORCH_CHECK(grad_residual.sizes() == input.sizes(), "grad_residual must have the input's shape");
  TORCH_CHECK(grad_weight.sizes() == weight.sizes(), "grad_weight must have the weight's shape");
  TORCH_CHECK(grad_post_weight.has_value() == post_weight.has_value(),
              "grad_post_weight and post_weight go together");
  TORCH_CHECK(grad_gate.has_value() == gate.has_value(), "grad_gate and gate go together");
  const Rows d = rows_arg(grad_out, "grad_out", c.hidden, input, type);
  const Rows t = rows_arg(residual_out, "residual", c.hidden, input, type);
  const Rows gi = rows_arg(grad_input, "grad_input", c.hidden, input, type);
  const Rows gr = rows_arg(grad_residual, "grad_residual", c.hidden, input, type);
  const Rows gw = rows_arg(grad_weight, "grad_weight", c.hidden, input, type);
  Rows e, gp, gg;
  if (grad_residual_out.has_value()) {
    TORCH_CHECK(grad_residual_out->sizes() == input.sizes(), "grad_residual must have the input's shape");
    e = rows_arg(*grad_residual_out, "grad_residual", c.hidden, input, type);
  }
  if (post_weight.has_value()) {
    TORCH_CHECK(grad_post_weight->dim() == 1, "grad_post_weight.dim() == 1");
    gp = rows_arg(*grad_post_weight, "grad_post_weight", c.hidden, input, type);
  }
  if (gate.has_value()) {
    TORCH_CHECK(grad_gate->sizes() == gate->sizes(), "grad_gate must have the gate's shape");
    gg = rows_arg(*grad_gate, "grad_gate", c.gate_width, input, type);
  }
  if (c.hidden == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_gated_add_rms_norm_backward(
        gi.p, gr.p, gp.p, gw.p, gg.p, d.p, e.p, c.x.p, t.p, c.p.p, c.w.p, c.g.p, c.rows, c.hidden,
        c.rows_per_gate, c.gate_width, gi.stride, gr.stride, gg.stride, d.stride, e.stride, c.x.stride,
        t.stride, c.g.stride, residual_scale, eps, c.dtype, ws, bytes, s, flags);
  });
}

float* float_out(const at::Tensor& t, const char* name, int64_t count, const at::Tensor& like) {
  return const_cast<float*>(float_rows(t, name, count, like));
}

void linear_log_probs(at::Tensor& log_prob, at::Tensor& entropy, at::Tensor& lse,
                      c10::optional<at::Tensor> top_log_probs, c10::optional<at::Tensor> top_indices,
                      const at::Tensor& input, const at::Tensor& weight, const at::Tensor& target,
                      double temperature, int64_t ignore_index) {
  const LossCall c = check_loss(input, weight, target);
  float* lp = float_out(log_prob, "log_prob", c.rows, input);
  float* hp = float_out(entropy, "entropy", c.rows, input);
  float* ep = float_out(lse, "lse", c.rows, input);
  TORCH_CHECK(top_log_probs.has_value() == top_indices.has_value(),
              "top_log_probs and top_indices go together");
  int64_t top = 0;
  float* vp = nullptr;
  int64_t* ip = nullptr;
  if (top_log_probs.has_value()) {
    TORCH_CHECK(top_log_probs->dim() >= 1 && top_indices->sizes() == top_log_probs->sizes(),
                "top_log_probs and top_indices must have one shape");
    top = top_log_probs->size(-1);
    TORCH_CHECK(top >= 1 && top <= 64 && top <= c.vocab, "top must be between 0 and 64 and at most vocab");
    TORCH_CHECK(top_indices->scalar_type() == at::kLong && top_indices->is_contiguous() &&
                    top_indices->is_cuda() && top_indices->device() == input.device(),
                "top_indices must be a contiguous int64 tensor");
    vp = float_out(*top_log_probs, "top_log_probs", c.rows * top, input);
    ip = top_indices->data_ptr<int64_t>();
  }
  if (c.rows == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_linear_log_probs(lp, hp, ep, vp, ip, c.x.p, c.w.p, c.target, ignore_index, temperature, top,
                                 c.rows, c.hidden, c.vocab, c.x.stride, c.w.stride, c.dtype, ws, bytes, s,
                                 flags);
  });
}

void linear_log_probs_backward(at::Tensor& grad_input, at::Tensor& grad_weight,
                               const at::Tensor& grad_log_prob, c10::optional<at::Tensor> grad_entropy,
                               const at::Tensor& input, const at::Tensor& weight,
                               const at::Tensor& target, const at::Tensor& lse,
                               c10::optional<at::Tensor> entropy, double temperature,
                               int64_t ignore_index) {
  const LossCall c = check_loss(input, weight, target);
  TORCH_CHECK(grad_input.sizes() == input.sizes(), "grad_input must have the input's shape");
  TORCH_CHECK(grad_weight.sizes() == weight.sizes(), "grad_weight must have the weight's shape");
  const Rows gi = rows_arg(grad_input, "grad_input", c.hidden, input, input.scalar_type());
  const Rows gw = rows_arg(grad_weight, "grad_weight", c.hidden, input, input.scalar_type());
  const float* gl = float_rows(grad_log_prob, "grad_log_prob", c.rows, input);
  const float* ep = float_rows(lse, "lse", c.rows, input);
  const float *ge = nullptr, *hp = nullptr;
  if (grad_entropy.has_value()) {
    TORCH_CHECK(entropy.has_value(), "grad_entropy needs the forward call's entropy");
    ge = float_rows(*grad_entropy, "grad_entropy", c.rows, input);
    hp = float_rows(*entropy, "entropy", c.rows, input);
  }
  if (c.hidden == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_linear_log_probs_backward(gi.p, gw.p, gl, ge, c.x.p, c.w.p, c.target, ep, hp, ignore_index,
                                          temperature, c.rows, c.hidden, c.vocab, gi.stride, gw.stride,
                                          c.x.stride, c.w.stride, c.dtype, ws, bytes, s, flags);
  });
}

void rms_norm_int8(at::Tensor& out, at::Tensor& scales, const at::Tensor& input,
                   c10::optional<at::Tensor> weight, c10::optional<at::Tensor> residual,
                   c10::optional<at::Tensor> residual_out, double eps) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  const int dtype = dtype_code(input);
  const int64_t hidden = input.size(-1), rows = leading(input);
  const at::ScalarType type = input.scalar_type();
  TORCH_CHECK(out.sizes() == input.sizes(), "out must have the input's shape");
  TORCH_CHECK(residual.has_value() || !residual_out.has_value(), "residual_out needs a residual");
  const Rows x = rows_arg(input, "input", hidden, input, type);
  const Rows q = rows_arg(out, "out", hidden, input, at::kChar);
  float* sp = float_out(scales, "scales", rows, input);
  Rows w, r, t;
  if (weight.has_value()) {
    TORCH_CHECK(weight->dim() == 1, "weight.dim() == 1");
    w = rows_arg(*weight, "weight", hidden, input, type);
  }
  if (residual.has_value()) {
    const at::Tensor& total = residual_out.has_value() ? *residual_out : *residual;
    TORCH_CHECK(residual->sizes() == input.sizes(), "residual must have the input's shape");
    TORCH_CHECK(total.sizes() == input.sizes(), "residual_out must have the input's shape");
    r = rows_arg(*residual, "residual", hidden, input, type);
    t = rows_arg(total, "residual_out", hidden, input, type);
  }
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(input.device().index()).stream();
  check_status(hprn_rms_norm_int8(static_cast<int8_t*>(q.p), sp, t.p, x.p, w.p, r.p, rows, hidden, q.stride,
                                  t.stride, x.stride, r.stride, eps, dtype, stream, HPRN_LAUNCH_DEFAULT));
}

void linear_int8(at::Tensor& out, const at::Tensor& input, const at::Tensor& input_scale,
                 const at::Tensor& weight, const at::Tensor& weight_scale, c10::optional<at::Tensor> bias) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 2, "weight must be [channels, hidden]");
  const int dtype = dtype_code(out);
  const int64_t hidden = input.size(-1), rows = leading(input), channels = weight.size(0);
  check_leading(out, "out", input);
  const Rows x = rows_arg(input, "input", hidden, input, at::kChar);
  const Rows w = rows_arg(weight, "weight", hidden, input, at::kChar);
  const Rows o = rows_arg(out, "out", channels, input, out.scalar_type());
  const float* xs = float_rows(input_scale, "input_scale", rows, input);
  const float* wsc = float_rows(weight_scale, "weight_scale", channels, input);
  Rows b;
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1, "bias.dim() == 1");
    b = rows_arg(*bias, "bias", channels, input, out.scalar_type());
  }
  if (rows == 0 || channels == 0) return;
  with_workspace(input, [&](void* ws, int64_t* bytes, cudaStream_t s, unsigned flags) {
    return hprn_linear_int8(o.p, static_cast<const int8_t*>(x.p), xs, static_cast<const int8_t*>(w.p), wsc, b.p,
                            rows, hidden, channels, o.stride, x.stride, w.stride, dtype, ws, bytes, s, flags);
  });
}

// The operators that make their outputs: a call from Python spends 2 to 5 us less on
// each than on a torch.empty of its own.

// What the shape-only kernels return, of whatever device and symbolic sizes.
struct Shapes {
  static at::Tensor dense_like(const at::Tensor& t, at::ScalarType type) {
    return at::empty_like(t, t.options().dtype(type), at::MemoryFormat::Contiguous);
  }
  static at::Tensor none(const at::Tensor& input) { return at::empty({0}, input.options()); }
  // The leading dimensions of `input`, and `last` after them where it is not negative.
  static at::Tensor rows_like(const at::Tensor& input, at::ScalarType type, int64_t last) {
    c10::SymDimVector sizes(input.sym_sizes().begin(), input.sym_sizes().end() - (input.dim() > 0));
    if (last >= 0) sizes.push_back(last);
    return at::empty_symint(sizes, input.options().dtype(type));
  }
  static at::Tensor product_like(const at::Tensor& input, const at::Tensor& weight, at::ScalarType type) {
    c10::SymDimVector sizes(input.sym_sizes().begin(), input.sym_sizes().end() - 1);
    sizes.push_back(weight.sym_size(0));
    return at::empty_symint(sizes, input.options().dtype(type));
  }
};

// The same on the input's GPU, past the dispatcher (0.6 us less a tensor).
struct Tensors {
  static at::Tensor make(c10::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, device, c10::nullopt));
  }
  static at::Tensor dense_like(const at::Tensor& t, at::ScalarType type) {
    // (What is on the host is refused where the arguments are checked.)
    return t.is_cuda() ? make(t.sizes(), type, t.device()) : Shapes::dense_like(t, type);
  }
  static at::Tensor none(const at::Tensor& input) { return make({0}, input.scalar_type(), input.device()); }
  static at::Tensor rows_like(const at::Tensor& input, at::ScalarType type, int64_t last) {
    c10::DimVector sizes(input.sizes().begin(), input.sizes().end() - (input.dim() > 0));
    if (last >= 0) sizes.push_back(last);
    return make(sizes, type, input.device());
  }
  static at::Tensor product_like(const at::Tensor& input, const at::Tensor& weight, at::ScalarType type) {
    return rows_like(input, type, weight.size(0));
  }
};

// The operators below fall through Autograd, whose own bookkeeping costs each call host
// time, so that the dispatcher does not tell a caller who asks for gradients: they do.
inline bool asks(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
inline bool asks(const c10::optional<at::Tensor>& t) { return t.has_value() && asks(*t); }
template <typename... Ts>
bool any_asks(const Ts&... t) {
  return c10::GradMode::is_enabled() && (asks(t) || ...);
}
#define HPRN_NOTE_NO_HISTORY(name, differentiable, ...)                                                        \
  if (any_asks(__VA_ARGS__))                                                                                   \
  TORCH_WARN_ONCE("hp_rms_norm::" name ": an input asks for gradients, but the outputs have no history and what " \
                  "is updated in place keeps none of it; " differentiable)

// Absent gradients are tensors without elements.
using BlockGrads = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

template <typename M>
BlockGrads block_grads_like(const at::Tensor& input, const c10::optional<at::Tensor>& post_weight,
                            const at::Tensor& weight, const c10::optional<at::Tensor>& gate) {
  auto like = [](const at::Tensor& t) { return M::dense_like(t, t.scalar_type()); };
  // (One each: outputs of an operator are not the same tensor.)
  auto like_or_none = [&](const c10::optional<at::Tensor>& t) {
    return t.has_value() ? like(*t) : M::none(input);
  };
  return {like(input), like(input), like_or_none(post_weight), like(weight), like_or_none(gate)};
}

BlockGrads gated_add_rms_norm_backward_new(const at::Tensor& grad_out, c10::optional<at::Tensor> grad_residual_out,
                                           const at::Tensor& input, const at::Tensor& residual_out,
                                           c10::optional<at::Tensor> post_weight, const at::Tensor& weight,
                                           c10::optional<at::Tensor> gate, double residual_scale, double eps) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  HPRN_NOTE_NO_HISTORY("gated_add_rms_norm_backward", "there are no second derivatives", grad_out, grad_residual_out, input, residual_out,
                       post_weight, weight, gate);
  BlockGrads grads = block_grads_like<Tensors>(input, post_weight, weight, gate);
  auto& [gi, gr, gp, gw, gg] = grads;
  if (gate.has_value() && input.numel() == 0) gg.zero_();  // a gate without rows
  c10::optional<at::Tensor> grad_post, grad_gate;
  if (post_weight.has_value()) grad_post = gp;
  if (gate.has_value()) grad_gate = gg;
  gated_add_rms_norm_backward(gi, gr, grad_post, gw, grad_gate, grad_out, grad_residual_out, input, residual_out,
                              post_weight, weight, gate, residual_scale, eps);
  return grads;
}

BlockGrads gated_add_rms_norm_backward_new_meta(const at::Tensor&, c10::optional<at::Tensor>, const at::Tensor& input,
                                                const at::Tensor&, c10::optional<at::Tensor> post_weight,
                                                const at::Tensor& weight, c10::optional<at::Tensor> gate, double,
                                                double) {
  return block_grads_like<Shapes>(input, post_weight, weight, gate);
}

using LogProbOutputs = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

template <typename M>
LogProbOutputs log_prob_outputs(const at::Tensor& input, int64_t top) {
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(top >= 0 && top <= 64, "top must be between 0 and 64 and at most vocab");
  auto rows = [&](at::ScalarType type, int64_t last) { return M::rows_like(input, type, last); };
  return {rows(at::kFloat, -1), rows(at::kFloat, -1), rows(at::kFloat, -1), rows(at::kFloat, top),
          rows(at::kLong, top)};
}

LogProbOutputs linear_log_probs_new(const at::Tensor& input, const at::Tensor& weight, const at::Tensor& target,
                                    int64_t top, double temperature, int64_t ignore_index) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  HPRN_NOTE_NO_HISTORY("linear_log_probs", "hp_rms_norm_b200.autograd has the differentiable form", input, weight);
  LogProbOutputs outputs = log_prob_outputs<Tensors>(input, top);
  auto& [log_prob, entropy, lse, values, indices] = outputs;
  c10::optional<at::Tensor> v, k;
  if (top > 0) v = values, k = indices;
  linear_log_probs(log_prob, entropy, lse, v, k, input, weight, target, temperature, ignore_index);
  return outputs;
}

LogProbOutputs linear_log_probs_new_meta(const at::Tensor& input, const at::Tensor&, const at::Tensor&, int64_t top,
                                         double, int64_t) {
  return log_prob_outputs<Shapes>(input, top);
}

std::tuple<at::Tensor, at::Tensor> linear_log_probs_backward_new(
    const at::Tensor& grad_log_prob, c10::optional<at::Tensor> grad_entropy, const at::Tensor& input,
    const at::Tensor& weight, const at::Tensor& target, const at::Tensor& lse, c10::optional<at::Tensor> entropy,
    double temperature, int64_t ignore_index) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  HPRN_NOTE_NO_HISTORY("linear_log_probs_backward", "there are no second derivatives", grad_log_prob, grad_entropy, input, weight, lse,
                       entropy);
  at::Tensor gi = Tensors::dense_like(input, input.scalar_type());
  at::Tensor gw = Tensors::dense_like(weight, weight.scalar_type());
  linear_log_probs_backward(gi, gw, grad_log_prob, grad_entropy, input, weight, target, lse, entropy, temperature,
                            ignore_index);
  return {gi, gw};
}

std::tuple<at::Tensor, at::Tensor> linear_log_probs_backward_new_meta(
    const at::Tensor&, c10::optional<at::Tensor>, const at::Tensor& input, const at::Tensor& weight,
    const at::Tensor&, const at::Tensor&, c10::optional<at::Tensor>, double, int64_t) {
  return {Shapes::dense_like(input, input.scalar_type()), Shapes::dense_like(weight, weight.scalar_type())};
}

template <typename M>
std::tuple<at::Tensor, at::Tensor> int8_outputs(const at::Tensor& input) {
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  return {M::dense_like(input, at::kChar), M::rows_like(input, at::kFloat, -1)};
}

std::tuple<at::Tensor, at::Tensor> rms_norm_int8_new(const at::Tensor& input, c10::optional<at::Tensor> weight,
                                                     c10::optional<at::Tensor> residual,
                                                     c10::optional<at::Tensor> residual_out, double eps) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  HPRN_NOTE_NO_HISTORY("rms_norm_int8", "8-bit integers have no gradients", input, weight, residual, residual_out);
  auto outputs = int8_outputs<Tensors>(input);
  rms_norm_int8(std::get<0>(outputs), std::get<1>(outputs), input, weight, residual, residual_out, eps);
  return outputs;
}

std::tuple<at::Tensor, at::Tensor> rms_norm_int8_sum(const at::Tensor& input, c10::optional<at::Tensor> weight,
                                                     const at::Tensor& residual, at::Tensor& residual_out,
                                                     double eps) {
  return rms_norm_int8_new(input, weight, residual, residual_out, eps);
}

std::tuple<at::Tensor, at::Tensor> rms_norm_int8_sum_meta(const at::Tensor& input, c10::optional<at::Tensor>,
                                                          const at::Tensor&, at::Tensor&, double) {
  return int8_outputs<Shapes>(input);
}

std::tuple<at::Tensor, at::Tensor> rms_norm_int8_new_meta(const at::Tensor& input, c10::optional<at::Tensor>,
                                                          c10::optional<at::Tensor>, c10::optional<at::Tensor>,
                                                          double) {
  return int8_outputs<Shapes>(input);
}

template <typename M>
at::Tensor int8_product_like(const at::Tensor& input, const at::Tensor& weight, at::ScalarType dtype) {
  TORCH_CHECK(input.dim() >= 1, "input.dim() >= 1");
  TORCH_CHECK(weight.dim() == 2, "weight must be [channels, hidden]");
  return M::product_like(input, weight, dtype);
}

at::Tensor linear_int8_new(const at::Tensor& input, const at::Tensor& input_scale, const at::Tensor& weight,
                           const at::Tensor& weight_scale, c10::optional<at::Tensor> bias, at::ScalarType dtype) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  HPRN_NOTE_NO_HISTORY("linear_int8", "8-bit integers have no gradients", input_scale, weight_scale, bias);
  at::Tensor out = int8_product_like<Tensors>(input, weight, dtype);
  linear_int8(out, input, input_scale, weight, weight_scale, bias);
  return out;
}

at::Tensor linear_int8_new_meta(const at::Tensor& input, const at::Tensor&, const at::Tensor& weight,
                                const at::Tensor&, c10::optional<at::Tensor>, at::ScalarType dtype) {
  return int8_product_like<Shapes>(input, weight, dtype);
}

void gated_add_rms_norm_meta(at::Tensor&, at::Tensor&, c10::optional<at::Tensor>, const at::Tensor&,
                             c10::optional<at::Tensor>, const at::Tensor&, c10::optional<at::Tensor>,
                             double, double) {}
void gated_add_rms_norm_sum_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                                 c10::optional<at::Tensor>, const at::Tensor&, c10::optional<at::Tensor>,
                                 double, double) {}
void rms_norm_int8_meta(at::Tensor&, at::Tensor&, const at::Tensor&, c10::optional<at::Tensor>,
                        c10::optional<at::Tensor>, c10::optional<at::Tensor>, double) {}
void linear_int8_meta(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                      const at::Tensor&, c10::optional<at::Tensor>) {}
void gated_linear_meta(at::Tensor&, c10::optional<at::Tensor>, const at::Tensor&, const at::Tensor&,
                       c10::string_view) {}
void gated_linear_backward_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                                const at::Tensor&, c10::optional<at::Tensor>, c10::string_view) {}
void linear_cross_entropy_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                               const at::Tensor&, int64_t) {}
void linear_cross_entropy_backward_meta(at::Tensor&, at::Tensor&, const at::Tensor&,
                                        const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                        const at::Tensor&, int64_t) {}
void rms_norm_backward_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, c10::optional<at::Tensor>, double) {}
void grad_norm_meta(at::Tensor&, at::TensorList) {}
void clip_grad_norm_meta(at::TensorList, at::Tensor&, at::TensorList, double) {}

// Shape-only kernels for tracing (torch.compile / FakeTensor): the ops return
// nothing and only mutate their annotated arguments.
void rms_norm_meta(at::Tensor&, const at::Tensor&, at::Tensor&, double) {}
void relu_meta(at::Tensor&, const at::Tensor&) {}
void rms_norm_out_meta(at::Tensor&, const at::Tensor&, const at::Tensor&,
                       c10::optional<at::Tensor>, double) {}
void rms_norm_fp8_meta(at::Tensor&, const at::Tensor&, const at::Tensor&,
                       c10::optional<at::Tensor>, double, c10::optional<at::Tensor>,
                       c10::optional<at::Tensor>) {}
void act_and_mul_meta(at::Tensor&, const at::Tensor&) {}
void rms_norm_nvfp4_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                         c10::optional<at::Tensor>, double, const at::Tensor&) {}
void rms_norm_fp8_group_meta(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                             c10::optional<at::Tensor>, double, int64_t, bool) {}

}  // namespace

TORCH_LIBRARY(hp_rms_norm, m) {
  // The reference's two operators.
  m.def("rms_norm(Tensor(a!) input, Tensor weight, Tensor(b!) residual, float eps) -> ()");
  m.def("relu(Tensor(a!) out, Tensor input) -> ()");
  // Extensions: plain / out-of-place RMSNorm and fp8-output RMSNorm.
  m.def("rms_norm_out(Tensor(a!) out, Tensor input, Tensor weight, Tensor(b!)? residual, "
        "float eps) -> ()");
  m.def("rms_norm_fp8(Tensor(a!) out, Tensor input, Tensor weight, Tensor(b!)? residual, "
        "float eps, Tensor? scale, Tensor(c!)? row_scales) -> ()");
  m.def("rms_norm_nvfp4(Tensor(a!) out, Tensor(b!) block_scales, Tensor input, Tensor weight, "
        "Tensor(c!)? residual, float eps, Tensor global_scale) -> ()");
  m.def("rms_norm_fp8_group(Tensor(a!) out, Tensor(b!) scales, Tensor input, Tensor weight, "
        "Tensor(c!)? residual, float eps, int group_size, bool scale_pow2) -> ()");
  // Extensions: gated activations.
  m.def("silu_and_mul(Tensor(a!) out, Tensor input) -> ()");
  m.def("gelu_and_mul(Tensor(a!) out, Tensor input) -> ()");
  m.def("gelu_tanh_and_mul(Tensor(a!) out, Tensor input) -> ()");
  // Extensions: training operators.
  m.def("gated_linear(Tensor(a!) out, Tensor(b!)? gate_up, Tensor input, Tensor weight, "
        "str act) -> ()");
  m.def("gated_linear_backward(Tensor(a!) grad_input, Tensor(b!) grad_weight, Tensor grad_out, "
        "Tensor input, Tensor weight, Tensor? gate_up, str act) -> ()");
  m.def("linear_cross_entropy(Tensor(a!) loss, Tensor(b!) lse, Tensor input, Tensor weight, "
        "Tensor target, int ignore_index) -> ()");
  m.def("linear_cross_entropy_backward(Tensor(a!) grad_input, Tensor(b!) grad_weight, "
        "Tensor grad_loss, Tensor input, Tensor weight, Tensor target, Tensor lse, "
        "int ignore_index) -> ()");
  m.def("rms_norm_backward(Tensor(a!) grad_input, Tensor(b!) grad_weight, Tensor grad_out, "
        "Tensor input, Tensor weight, Tensor? grad_residual, float eps) -> ()");
  m.def("gated_add_rms_norm(Tensor(a!) out, Tensor(b!) residual, Tensor(c!)? residual_out, Tensor input, "
        "Tensor? post_weight, Tensor weight, Tensor? gate, float residual_scale, float eps) -> ()");
  // The _sum forms leave residual as it is, so that a traced graph orders no write to it.
  // (Names of their own: overloads would fit the same calls by position.)
  m.def("gated_add_rms_norm_sum(Tensor(a!) out, Tensor(b!) residual_out, Tensor input, Tensor residual, "
        "Tensor? post_weight, Tensor weight, Tensor? gate, float residual_scale, float eps) -> ()");
  // (Gradients of what is absent come back without elements, as do alternatives with top 0.)
  m.def("gated_add_rms_norm_backward(Tensor grad_out, Tensor? grad_residual_out, Tensor input, "
        "Tensor residual_out, Tensor? post_weight, Tensor weight, Tensor? gate, float residual_scale, "
        "float eps) -> (Tensor grad_input, Tensor grad_residual, Tensor grad_post_weight, "
        "Tensor grad_weight, Tensor grad_gate)");
  m.def("linear_log_probs(Tensor input, Tensor weight, Tensor target, int top, float temperature, "
        "int ignore_index) -> (Tensor log_prob, Tensor entropy, Tensor lse, Tensor top_log_probs, "
        "Tensor top_indices)");
  m.def("linear_log_probs_backward(Tensor grad_log_prob, Tensor? grad_entropy, Tensor input, Tensor weight, "
        "Tensor target, Tensor lse, Tensor? entropy, float temperature, int ignore_index) -> "
        "(Tensor grad_input, Tensor grad_weight)");
  // Extensions: 8-bit integers.
  m.def("rms_norm_int8(Tensor input, Tensor? weight, Tensor(a!)? residual, Tensor(b!)? residual_out, "
        "float eps) -> (Tensor codes, Tensor scales)");
  m.def("rms_norm_int8_sum(Tensor input, Tensor? weight, Tensor residual, Tensor(a!) residual_out, "
        "float eps) -> (Tensor codes, Tensor scales)");
  m.def("rms_norm_int8.out(Tensor(a!) out, Tensor(b!) scales, Tensor input, Tensor? weight, "
        "Tensor(c!)? residual, Tensor(d!)? residual_out, float eps) -> ()");
  m.def("linear_int8(Tensor input, Tensor input_scale, Tensor weight, Tensor weight_scale, Tensor? bias, "
        "ScalarType dtype) -> Tensor");
  m.def("linear_int8.out(Tensor(a!) out, Tensor input, Tensor input_scale, Tensor weight, "
        "Tensor weight_scale, Tensor? bias) -> ()");
  m.def("grad_norm(Tensor(a!) norm, Tensor[] grads) -> ()");
  m.def("clip_grad_norm(Tensor(a!)[] out, Tensor(b!) norm, Tensor[] grads, float max_norm) -> ()");
}

TORCH_LIBRARY_IMPL(hp_rms_norm, CUDA, m) {
  m.impl("rms_norm", &rms_norm);
  m.impl("relu", &relu);
  m.impl("rms_norm_out", &rms_norm_out);
  m.impl("rms_norm_fp8", &rms_norm_fp8);
  m.impl("rms_norm_nvfp4", &rms_norm_nvfp4);
  m.impl("rms_norm_fp8_group", &rms_norm_fp8_group);
  m.impl("silu_and_mul", &silu_and_mul);
  m.impl("gelu_and_mul", &gelu_and_mul);
  m.impl("gelu_tanh_and_mul", &gelu_tanh_and_mul);
  m.impl("gated_linear", &gated_linear);
  m.impl("gated_linear_backward", &gated_linear_backward);
  m.impl("linear_cross_entropy", &linear_cross_entropy);
  m.impl("linear_cross_entropy_backward", &linear_cross_entropy_backward);
  m.impl("rms_norm_backward", &rms_norm_backward);
  m.impl("grad_norm", &grad_norm);
  m.impl("clip_grad_norm", &clip_grad_norm);
  m.impl("gated_add_rms_norm", &gated_add_rms_norm);
  m.impl("gated_add_rms_norm_sum", &gated_add_rms_norm_sum);
  m.impl("gated_add_rms_norm_backward", &gated_add_rms_norm_backward_new);
  m.impl("linear_log_probs", &linear_log_probs_new);
  m.impl("linear_log_probs_backward", &linear_log_probs_backward_new);
  m.impl("rms_norm_int8", &rms_norm_int8_new);
  m.impl("rms_norm_int8_sum", &rms_norm_int8_sum);
  m.impl("rms_norm_int8.out", &rms_norm_int8);
  m.impl("linear_int8", &linear_int8_new);
  m.impl("linear_int8.out", &linear_int8);
}

TORCH_LIBRARY_IMPL(hp_rms_norm, Meta, m) {
  m.impl("rms_norm", &rms_norm_meta);
  m.impl("relu", &relu_meta);
  m.impl("rms_norm_out", &rms_norm_out_meta);
  m.impl("rms_norm_fp8", &rms_norm_fp8_meta);
  m.impl("rms_norm_nvfp4", &rms_norm_nvfp4_meta);
  m.impl("rms_norm_fp8_group", &rms_norm_fp8_group_meta);
  m.impl("silu_and_mul", &act_and_mul_meta);
  m.impl("gelu_and_mul", &act_and_mul_meta);
  m.impl("gelu_tanh_and_mul", &act_and_mul_meta);
  m.impl("gated_linear", &gated_linear_meta);
  m.impl("gated_linear_backward", &gated_linear_backward_meta);
  m.impl("linear_cross_entropy", &linear_cross_entropy_meta);
  m.impl("linear_cross_entropy_backward", &linear_cross_entropy_backward_meta);
  m.impl("rms_norm_backward", &rms_norm_backward_meta);
  m.impl("grad_norm", &grad_norm_meta);
  m.impl("clip_grad_norm", &clip_grad_norm_meta);
  m.impl("gated_add_rms_norm", &gated_add_rms_norm_meta);
  m.impl("gated_add_rms_norm_sum", &gated_add_rms_norm_sum_meta);
  m.impl("gated_add_rms_norm_backward", &gated_add_rms_norm_backward_new_meta);
  m.impl("linear_log_probs", &linear_log_probs_new_meta);
  m.impl("linear_log_probs_backward", &linear_log_probs_backward_new_meta);
  m.impl("rms_norm_int8", &rms_norm_int8_new_meta);
  m.impl("rms_norm_int8_sum", &rms_norm_int8_sum_meta);
  m.impl("rms_norm_int8.out", &rms_norm_int8_meta);
  m.impl("linear_int8", &linear_int8_new_meta);
  m.impl("linear_int8.out", &linear_int8_meta);
}

// No gradients of their own (hp_rms_norm_b200.autograd has the differentiable forms):
// outputs of these have no history, whatever their inputs ask for, and a call that such
// an input reaches says so once (HPRN_NOTE_NO_HISTORY).
TORCH_LIBRARY_IMPL(hp_rms_norm, Autograd, m) {
  m.impl("gated_add_rms_norm_backward", torch::CppFunction::makeFallthrough());
  m.impl("linear_log_probs", torch::CppFunction::makeFallthrough());
  m.impl("linear_log_probs_backward", torch::CppFunction::makeFallthrough());
  m.impl("rms_norm_int8", torch::CppFunction::makeFallthrough());
  m.impl("rms_norm_int8_sum", torch::CppFunction::makeFallthrough());
  m.impl("linear_int8", torch::CppFunction::makeFallthrough());
}
