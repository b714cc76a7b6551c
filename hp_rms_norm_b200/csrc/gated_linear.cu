// A gated linear layer, the first half of a SwiGLU / GeGLU feed-forward block:
//   G = X Wg^T,  U = X Wu^T,  out = act(G) * U
// with X [rows, hidden] and weight = [Wg; Wu] of 2d rows of `hidden`, both
// products, the activation and the product of the two in one kernel: a CTA
// computes the gate and the up columns of the same outputs, so G and U meet in
// its accumulators and only `out` (d columns) is written.  A training pass
// may also have G and U, in fp32, written to `gate_up` for the backward pass.
//
// Backward, D the gradient of out:
//   dU = D act(G),  dG = D U act'(G),  S = [dG | dU] (16-bit, [rows, 2d])
//   dX = S weight,  dW = S^T X
// S is what the tensor cores read, so its rounding to 16 bits is the one
// rounding between the inputs and the fp32 sums of dX and dW.  G and U come
// from `gate_up`, or are computed again (4 rows hidden d more operations, no
// 8 rows d bytes kept).
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "gated.cuh"
#include "matmul.cuh"
#include "runtime.cuh"

namespace hprn {

template <typename T, int ACT>
struct GatedEpilogue {
  static constexpr bool kPaired = true;
  uint16_t* out = nullptr;
  int64_t ld = 0;
  int64_t d = 0;
  float* gate_up = nullptr;  // or null
  int64_t gate_up_ld = 0;

  struct Row {};
  __device__ __forceinline__ Row begin(int64_t) const { return {}; }
  __device__ __forceinline__ void chunk(Row&, int64_t i, int64_t j, const float (&g)[kChunk],
                                        const float (&u)[kChunk]) const {
    if (gate_up) {
      store_chunk_f32(gate_up + i * gate_up_ld, j, d, g);
      store_chunk_f32(gate_up + i * gate_up_ld + d, j, d, u);
    }
    float h[kChunk];
#pragma unroll
    for (int k = 0; k < kChunk; ++k) h[k] = activate_with_slope<ACT>(g[k]).value * u[k];
    store_chunk<T>(out + i * ld, j, d, h);
  }
  __device__ __forceinline__ void end(Row&, int64_t, int64_t) const {}
};

// S's chunk from the same chunk of G, U and D.
template <typename T, int ACT>
__device__ __forceinline__ void gated_gradients(float (&g)[kChunk], float (&u)[kChunk],
                                                const float (&dout)[kChunk]) {
#pragma unroll
  for (int k = 0; k < kChunk; ++k) {
    const ActValue a = activate_with_slope<ACT>(g[k]);
    g[k] = dout[k] * u[k] * a.slope;
    u[k] = dout[k] * a.value;
  }
}

template <typename T>
__device__ __forceinline__ void load_chunk(const uint16_t* row, int64_t j, int64_t n,
                                           float (&v)[kChunk]) {
  const uint16_t* p = row + j;
  if (j + kChunk <= n && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int h = 0; h < kChunk / 8; ++h) {
      const uint4 q = reinterpret_cast<const uint4*>(p)[h];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2<T>(w[k]);
        v[8 * h + 2 * k] = f.x, v[8 * h + 2 * k + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) v[k] = j + k < n ? unpack1<T>(p[k]) : 0.f;
  }
}

// The gradient S where G and U are computed again.
template <typename T, int ACT>
struct GatedGradEpilogue {
  static constexpr bool kPaired = true;
  const uint16_t* dout = nullptr;
  int64_t dout_ld = 0;
  uint16_t* s = nullptr;
  int64_t s_ld = 0;
  int64_t d = 0;

  struct Row {};
  __device__ __forceinline__ Row begin(int64_t) const { return {}; }
  __device__ __forceinline__ void chunk(Row&, int64_t i, int64_t j, const float (&g)[kChunk],
                                        const float (&u)[kChunk]) const {
    float dg[kChunk], du[kChunk], o[kChunk];
    load_chunk<T>(dout + i * dout_ld, j, d, o);
#pragma unroll
    for (int k = 0; k < kChunk; ++k) dg[k] = g[k], du[k] = u[k];
    gated_gradients<T, ACT>(dg, du, o);
    store_chunk<T>(s + i * s_ld, j, d, dg);
    store_chunk<T>(s + i * s_ld + d, j, d, du);
  }
  __device__ __forceinline__ void end(Row&, int64_t, int64_t) const {}
};

// S from a kept gate_up.  Memory-bound: 14 bytes per output element.
struct GatedGradArgs {
  const uint16_t* dout;
  int64_t dout_ld;
  const float* gate_up;
  int64_t gate_up_ld;
  uint16_t* s;
  int64_t s_ld;
  int64_t rows, d;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_grad_rows(GatedGradArgs a) {
  pdl_wait();
  const int64_t n = a.rows * a.d;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n; e += step) {
    const int64_t i = e / a.d, j = e - i * a.d;
    const float g = a.gate_up[i * a.gate_up_ld + j], u = a.gate_up[i * a.gate_up_ld + a.d + j];
    const float o = unpack1<T>(a.dout[i * a.dout_ld + j]);
    const ActValue v = activate_with_slope<ACT>(g);
    a.s[i * a.s_ld + j] = pack1<T>(o * u * v.slope);
    a.s[i * a.s_ld + a.d + j] = pack1<T>(o * v.value);
  }
}

namespace {

// Calls f(T{}, integral_constant<int, act>).
template <typename F>
int with_type_and_act(int dtype, int act, F&& f) {
  auto with_act = [&](auto t) {
    switch (act) {
      case HPRN_ACT_SILU: return f(t, std::integral_constant<int, HPRN_ACT_SILU>{});
      case HPRN_ACT_GELU: return f(t, std::integral_constant<int, HPRN_ACT_GELU>{});
      default: return f(t, std::integral_constant<int, HPRN_ACT_GELU_TANH>{});
    }
  };
  return dtype == HPRN_DTYPE_BF16 ? with_act(__nv_bfloat16{}) : with_act(__half{});
}

int check_common(int64_t rows, int64_t hidden, int64_t d, int act, int dtype, unsigned flags,
                 const int64_t* workspace_bytes) {
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (act != HPRN_ACT_SILU && act != HPRN_ACT_GELU && act != HPRN_ACT_GELU_TANH)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown activation");
  if (rows < 0 || hidden < 0 || d < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || hidden > kMaxExtent || d > kMaxExtent / 2)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows, hidden and 2d must be at most 2^30");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  return HPRN_OK;
}

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_gated_linear(void* out, float* gate_up, const void* input, const void* weight,
                      int64_t rows, int64_t hidden, int64_t d, int64_t out_row_stride,
                      int64_t gate_up_row_stride, int64_t input_row_stride,
                      int64_t weight_row_stride, int act, int dtype, void* workspace,
                      int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  int st = check_common(rows, hidden, d, act, dtype, flags, workspace_bytes);
  if (st != HPRN_OK) return st;
  if ((rows > 1 && (out_row_stride < d || input_row_stride < hidden ||
                    (gate_up && gate_up_row_stride < 2 * d))) ||
      (d > 0 && weight_row_stride < hidden))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  Workspace ws(workspace, *workspace_bytes);
  const AlignedRows x(ws, input, rows, hidden, input_row_stride);
  const AlignedRows w(ws, weight, 2 * d, hidden, weight_row_stride);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (rows == 0 || d == 0) return ok();
  if (!out || (hidden > 0 && (!input || !weight)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(out, 2) || !aligned(input, 2) || !aligned(weight, 2) || !aligned(gate_up, 4))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(out, rows, d, out_row_stride),
                       extent32(gate_up, rows, 2 * d, gate_up_row_stride)};
  const Extent ins[] = {extent16(input, rows, hidden, input_row_stride),
                      extent16(weight, 2 * d, hidden, weight_row_stride)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if ((st = x.prepare(cs, flags)) != HPRN_OK || (st = w.prepare(cs, flags)) != HPRN_OK) return st;
  Product q;
  q.a = {x.data(), x.ld()};
  q.b = {w.data(), w.ld()};
  q.m = rows, q.n = d, q.depth = hidden, q.pair_offset = d;
  return with_type_and_act(dtype, act, [&](auto t, auto a) {
    using T = decltype(t);
    GatedEpilogue<T, decltype(a)::value> e;
    e.out = static_cast<uint16_t*>(out), e.ld = out_row_stride, e.d = d;
    e.gate_up = gate_up, e.gate_up_ld = gate_up_row_stride;
    return launch_product<T, true, true>(q, e, cs, flags, "gated_linear");
  });
}

int hprn_gated_linear_backward(void* grad_input, void* grad_weight, const void* grad_out,
                               const float* gate_up, const void* input, const void* weight,
                               int64_t rows, int64_t hidden, int64_t d,
                               int64_t grad_input_row_stride, int64_t grad_weight_row_stride,
                               int64_t grad_out_row_stride, int64_t gate_up_row_stride,
                               int64_t input_row_stride, int64_t weight_row_stride, int act,
                               int dtype, void* workspace, int64_t* workspace_bytes, void* stream,
                               unsigned flags) {
  using namespace hprn;
  int st = check_common(rows, hidden, d, act, dtype, flags, workspace_bytes);
  if (st != HPRN_OK) return st;
  if ((rows > 1 && (grad_out_row_stride < d || input_row_stride < hidden ||
                    grad_input_row_stride < hidden || (gate_up && gate_up_row_stride < 2 * d))) ||
      (d > 0 && (weight_row_stride < hidden || grad_weight_row_stride < hidden)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  Workspace ws(workspace, *workspace_bytes);
  const AlignedRows x(ws, input, rows, hidden, input_row_stride);
  const AlignedRows w(ws, weight, 2 * d, hidden, weight_row_stride);
  const int64_t s_ld = round_up(2 * d, 16);
  uint16_t* s = ws.take<uint16_t>(rows * s_ld);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if ((rows > 0 && (!grad_input || !input)) || (d > 0 && (!grad_weight || !weight)) ||
      (rows > 0 && d > 0 && !grad_out))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(grad_input, 2) || !aligned(grad_weight, 2) || !aligned(grad_out, 2) ||
      !aligned(input, 2) || !aligned(weight, 2) || !aligned(gate_up, 4))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                       extent16(grad_weight, 2 * d, hidden, grad_weight_row_stride)};
  const Extent ins[] = {extent16(grad_out, rows, d, grad_out_row_stride),
                      extent32(gate_up, rows, 2 * d, gate_up_row_stride),
                      extent16(input, rows, hidden, input_row_stride),
                      extent16(weight, 2 * d, hidden, weight_row_stride)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if ((st = x.prepare(cs, flags)) != HPRN_OK || (st = w.prepare(cs, flags)) != HPRN_OK) return st;
  if (rows > 0 && d > 0) {
    st = with_type_and_act(dtype, act, [&](auto t, auto a) {
      using T = decltype(t);
      constexpr int kAct = decltype(a)::value;
      if (gate_up) {
        GatedGradArgs g{static_cast<const uint16_t*>(grad_out), grad_out_row_stride, gate_up,
                        gate_up_row_stride, s, s_ld, rows, d};
        const int64_t ctas = (rows * d + 1023) / 1024;
        const int64_t most = 16 * dev->sm_count;
        return launch_rows(gated_grad_rows<T, kAct>, dim3(static_cast<unsigned>(ctas < most ? ctas : most)),
                           dim3(256), cs, flags, "gated_linear_backward", g);
      }
      Product q;
      q.a = {x.data(), x.ld()};
      q.b = {w.data(), w.ld()};
      q.m = rows, q.n = d, q.depth = hidden, q.pair_offset = d;
      GatedGradEpilogue<T, kAct> e;
      e.dout = static_cast<const uint16_t*>(grad_out), e.dout_ld = grad_out_row_stride;
      e.s = s, e.s_ld = s_ld, e.d = d;
      return launch_product<T, true, true>(q, e, cs, flags, "gated_linear_backward");
    });
    if (st != HPRN_OK) return st;
  }
  // Without rows the weight's gradient is zero, without columns the input's:
  // sums of depth 0.
  auto gradients = [&](auto t) {
    using T = decltype(t);
    int r = HPRN_OK;
    if (rows > 0) {
      Product q;
      q.a = {s, s_ld};
      q.b = {w.data(), w.ld()};
      q.m = rows, q.n = hidden, q.depth = 2 * d;
      StoreEpilogue<T> e;
      e.out = static_cast<uint16_t*>(grad_input), e.ld = grad_input_row_stride, e.n = hidden;
      r = launch_product<T, true, false>(q, e, cs, flags, "gated_linear_backward");
    }
    if (r == HPRN_OK && d > 0) {
      Product q;
      q.a = {s, s_ld};
      q.b = {x.data(), x.ld()};
      q.m = 2 * d, q.n = hidden, q.depth = rows;
      StoreEpilogue<T> e;
      e.out = static_cast<uint16_t*>(grad_weight), e.ld = grad_weight_row_stride, e.n = hidden;
      r = launch_product<T, false, false>(q, e, cs, flags, "gated_linear_backward");
    }
    return r;
  };
  return dtype == HPRN_DTYPE_BF16 ? gradients(__nv_bfloat16{}) : gradients(__half{});
}

}  // extern "C"
