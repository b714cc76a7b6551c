// Gradients of RMSNorm, y_j = x_j w_j inv, inv = rsqrt(mean(x^2) + eps), for a
// gradient D of y, with n_j = x_j inv:
//   dx_j = inv (w_j D_j - n_j mean_k(w_k D_k n_k)) [+ E_j]
//   dw_j = sum over rows of D_j n_j
// E is the gradient that reaches x another way: in a pre-norm block x is the
// updated residual, which the next layer reads as well.  For the fused add
// (residual += input; y = RMSNorm(residual) w) x is the updated residual and
// dx is the gradient of both the input and the residual.
//
// All sums are fp32; dx and dw are rounded to 16 bits once.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

struct NormGradArgs {
  uint16_t* dx;
  uint16_t* dw;
  const uint16_t* dy;
  const uint16_t* x;
  const uint16_t* w;
  const uint16_t* extra;  // E, or null
  int64_t rows, hidden;
  int64_t dx_stride, dy_stride, x_stride, extra_stride;
  float eps;
  float2* stats;   // per row: {inv, mean_k(w_k D_k n_k)}
  float* partial;  // [groups, hidden]: dw's sums over a group's rows
  int64_t groups;
};

__device__ __forceinline__ float2 block_sum(float2 v) {
  __shared__ float2 part[32];
  const int warps = blockDim.x / 32;
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(~0u, v.x, o);
    v.y += __shfl_xor_sync(~0u, v.y, o);
  }
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int k = 0; k < warps; ++k) s.x += part[k].x, s.y += part[k].y;
  return s;
}

// One CTA per row: the row's two sums.
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_stats(NormGradArgs a) {
  pdl_wait();
  const int64_t i = blockIdx.x;
  const uint16_t* x = a.x + i * a.x_stride;
  const uint16_t* dy = a.dy + i * a.dy_stride;
  float2 s = make_float2(0.f, 0.f);
  for (int64_t j = threadIdx.x; j < a.hidden; j += blockDim.x) {
    const float v = unpack1<T>(x[j]);
    s.x = fmaf(v, v, s.x);
    s.y = fmaf(unpack1<T>(a.w[j]) * unpack1<T>(dy[j]), v, s.y);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) {
    const float inv = rsqrtf(s.x / static_cast<float>(a.hidden) + a.eps);
    a.stats[i] = make_float2(inv, s.y * inv / static_cast<float>(a.hidden));
  }
}

// A group of rows x blockDim columns per CTA: dx, and the group's part of dw.
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_columns(NormGradArgs a) {
  pdl_wait();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (j >= a.hidden) return;
  const float w = unpack1<T>(a.w[j]);
  float sum = 0.f;
  for (int64_t i = blockIdx.y; i < a.rows; i += a.groups) {
    const float2 st = a.stats[i];
    const float n = unpack1<T>(a.x[i * a.x_stride + j]) * st.x;
    const float d = unpack1<T>(a.dy[i * a.dy_stride + j]);
    sum = fmaf(d, n, sum);
    float g = st.x * (w * d - n * st.y);
    if (a.extra) g += unpack1<T>(a.extra[i * a.extra_stride + j]);
    a.dx[i * a.dx_stride + j] = pack1<T>(g);
  }
  a.partial[blockIdx.y * a.hidden + j] = sum;
}

template <typename T>
__global__ void __launch_bounds__(256) norm_grad_weight(NormGradArgs a) {
  pdl_wait();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (j >= a.hidden) return;
  float sum = 0.f;
  for (int64_t g = 0; g < a.groups; ++g) sum += a.partial[g * a.hidden + j];
  a.dw[j] = pack1<T>(sum);
}

template <typename T>
int launch_norm_grad(const NormGradArgs& a, cudaStream_t stream, unsigned flags) {
  const char* what = "rms_norm_backward";
  const unsigned cols = static_cast<unsigned>((a.hidden + 255) / 256);
  if (a.rows > 0) {
    int st = launch_rows(norm_grad_stats<T>, dim3(static_cast<unsigned>(a.rows)), dim3(256), stream, flags,
                         what, a);
    if (st != HPRN_OK) return st;
    st = launch_rows(norm_grad_columns<T>, dim3(cols, static_cast<unsigned>(a.groups)), dim3(256), stream,
                     flags, what, a);
    if (st != HPRN_OK) return st;
  }
  return launch_rows(norm_grad_weight<T>, dim3(cols), dim3(256), stream, flags, what, a);
}

}  // namespace hprn

extern "C" int hprn_rms_norm_backward(void* grad_input, void* grad_weight, const void* grad_out,
                                      const void* input, const void* weight,
                                      const void* grad_residual, int64_t rows, int64_t hidden,
                                      int64_t grad_input_row_stride, int64_t grad_out_row_stride,
                                      int64_t input_row_stride, int64_t grad_residual_row_stride,
                                      double eps, int dtype, void* workspace,
                                      int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (rows < 0 || hidden < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || hidden > kMaxExtent)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows and hidden must be at most 2^30");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  if (rows > 1 && (grad_input_row_stride < hidden || grad_out_row_stride < hidden ||
                   input_row_stride < hidden || (grad_residual && grad_residual_row_stride < hidden)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  NormGradArgs a{};
  a.groups = rows < 64 ? rows : 64;
  Workspace ws(workspace, *workspace_bytes);
  a.stats = ws.take<float2>(rows);
  a.partial = ws.take<float>(a.groups * hidden);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if (!grad_weight || !weight || (rows > 0 && (!grad_input || !grad_out || !input)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(grad_input, 2) || !aligned(grad_weight, 2) || !aligned(grad_out, 2) ||
      !aligned(input, 2) || !aligned(weight, 2) || !aligned(grad_residual, 2))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                       extent16(grad_weight, 1, hidden, hidden)};
  const Extent ins[] = {extent16(grad_out, rows, hidden, grad_out_row_stride),
                      extent16(input, rows, hidden, input_row_stride), extent16(weight, 1, hidden, hidden),
                      extent16(grad_residual, rows, hidden, grad_residual_row_stride)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  a.dx = static_cast<uint16_t*>(grad_input), a.dw = static_cast<uint16_t*>(grad_weight);
  a.dy = static_cast<const uint16_t*>(grad_out), a.x = static_cast<const uint16_t*>(input);
  a.w = static_cast<const uint16_t*>(weight), a.extra = static_cast<const uint16_t*>(grad_residual);
  a.rows = rows, a.hidden = hidden;
  a.dx_stride = grad_input_row_stride, a.dy_stride = grad_out_row_stride;
  a.x_stride = input_row_stride, a.extra_stride = grad_residual_row_stride;
  a.eps = static_cast<float>(eps);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == HPRN_DTYPE_BF16 ? launch_norm_grad<__nv_bfloat16>(a, cs, flags)
                                  : launch_norm_grad<__half>(a, cs, flags);
}
