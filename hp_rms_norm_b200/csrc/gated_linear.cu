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
// 8 rows d bytes kept): 4096 x 4096 x 2 * 14336 bf16, backward 1536 us with the
// products kept, 2195 without, forward 648 us writing them, 590 without.
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
  static constexpr int kSegment = 0;
  Out16 out;
  Out32 gate, up;  // null to leave out

  struct Row {};
  __device__ __forceinline__ Row begin(const Lane&, int64_t) const { return {}; }
  __device__ __forceinline__ void chunk(Row&, const Lane& l, int64_t i, int64_t j, float (&g)[kChunk],
                                        float (&u)[kChunk]) const {
    if (gate.p) {
      gate.store(l, i, j, g);
      up.store(l, i, j, u);
    }
#pragma unroll
    for (int k = 0; k < kChunk; ++k) u[k] *= activate_with_slope<ACT>(g[k]).value;
    out.template store<T>(l, i, j, u);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
  __device__ __forceinline__ void point(int64_t i, int64_t j, float g, float u) const {
    if (gate.p) gate.p[i * gate.ld + j] = g, up.p[i * up.ld + j] = u;
    out.p[i * out.ld + j] = pack1<T>(activate_with_slope<ACT>(g).value * u);
  }
};

// [dG | dU] in place of G and U, for the gradient D of act(G) U.
template <int ACT, int N>
__device__ __forceinline__ void gated_gradients(float (&g)[N], float (&u)[N], const float (&dout)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const ActValue a = activate_with_slope<ACT>(g[k]);
    g[k] = dout[k] * u[k] * a.slope;
    u[k] = dout[k] * a.value;
  }
}

// The gradient S where G and U are computed again.
template <typename T, int ACT>
struct GatedGradEpilogue {
  static constexpr bool kPaired = true;
  static constexpr int kSegment = 0;
  const uint16_t* dout = nullptr;
  int64_t dout_ld = 0;
  bool dout_aligned = false;  // every row to 16 bytes
  Out16 gate, up;

  struct Row {};
  __device__ __forceinline__ Row begin(const Lane&, int64_t) const { return {}; }
  __device__ __forceinline__ void chunk(Row&, const Lane& l, int64_t i, int64_t j, float (&g)[kChunk],
                                        float (&u)[kChunk]) const {
    float o[kChunk] = {};
    if (l.inside) {
      const uint16_t* p = dout + i * dout_ld + j;
      if (dout_aligned && j + kChunk <= gate.n) {
#pragma unroll
        for (int h = 0; h < kChunk / 8; ++h) {
          const uint4 q = reinterpret_cast<const uint4*>(p)[h];
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = unpack2<T>(w[k]);
            o[8 * h + 2 * k] = f.x, o[8 * h + 2 * k + 1] = f.y;
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < kChunk; ++k)
          if (j + k < gate.n) o[k] = unpack1<T>(p[k]);
      }
    }
    gated_gradients<ACT>(g, u, o);
    gate.template store<T>(l, i, j, g);
    up.template store<T>(l, i, j, u);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
  __device__ __forceinline__ void point(int64_t i, int64_t j, float gi, float ui) const {
    float g[1] = {gi}, u[1] = {ui}, o[1] = {unpack1<T>(dout[i * dout_ld + j])};
    gated_gradients<ACT>(g, u, o);
    gate.p[i * gate.ld + j] = pack1<T>(g[0]);
    up.p[i * up.ld + j] = pack1<T>(u[0]);
  }
};

// S from a kept gate_up.  Memory-bound: 14 bytes per output element.  Eight
// elements a thread where every row of every tensor starts on a 16-byte
// boundary and d is a multiple of 8.
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
__global__ void __launch_bounds__(256) gated_grad_vectors(GatedGradArgs a) {
  pdl_wait();
  const int64_t per_row = a.d / 8, n = a.rows * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const uint64_t pol = policy_evict_first();
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n; e += step) {
    const int64_t i = e / per_row, j = (e - i * per_row) * 8;
    const float* gp = a.gate_up + i * a.gate_up_ld + j;
    uint16_t* sp = a.s + i * a.s_ld + j;
    const Vec<16> g0 = ld_stream<16>(gp, pol), g1 = ld_stream<16>(gp + 4, pol);
    const Vec<16> u0 = ld_stream<16>(gp + a.d, pol), u1 = ld_stream<16>(gp + a.d + 4, pol);
    const Vec<16> d0 = ld_stream<16>(a.dout + i * a.dout_ld + j, pol);
    float g[8], u[8], o[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      g[k] = __uint_as_float(g0.w[k]), g[k + 4] = __uint_as_float(g1.w[k]);
      u[k] = __uint_as_float(u0.w[k]), u[k + 4] = __uint_as_float(u1.w[k]);
      const float2 f = unpack2<T>(d0.w[k]);
      o[2 * k] = f.x, o[2 * k + 1] = f.y;
    }
    gated_gradients<ACT>(g, u, o);
    Vec<16> sg, su;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sg.w[k] = pack2<T>(g[2 * k], g[2 * k + 1]);
      su.w[k] = pack2<T>(u[2 * k], u[2 * k + 1]);
    }
    st_global<16>(sp, sg);
    st_global<16>(sp + a.d, su);
  }
}

// The same for any alignment: a CTA takes 1024 columns of a row, four a thread.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_grad_elements(GatedGradArgs a) {
  constexpr int N = 4;
  pdl_wait();
  const int64_t per_row = (a.d + 1023) / 1024, n = a.rows * per_row;
  for (int64_t c = blockIdx.x; c < n; c += gridDim.x) {
    const int64_t i = c / per_row, j0 = (c - i * per_row) * 1024 + threadIdx.x;
    const float* gp = a.gate_up + i * a.gate_up_ld;
    const uint16_t* dp = a.dout + i * a.dout_ld;
    uint16_t* sp = a.s + i * a.s_ld;
    float g[N], u[N], o[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t j = j0 + k * 256;
      g[k] = u[k] = o[k] = 0.f;
      if (j < a.d) g[k] = gp[j], u[k] = gp[a.d + j], o[k] = unpack1<T>(dp[j]);
    }
    gated_gradients<ACT>(g, u, o);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t j = j0 + k * 256;
      if (j < a.d) sp[j] = pack1<T>(g[k]), sp[a.d + j] = pack1<T>(u[k]);
    }
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
  const AlignedRows x(ws, input, rows, hidden, input_row_stride, 2 * d);
  const AlignedRows w(ws, weight, 2 * d, hidden, weight_row_stride, rows);
  const PlannedProduct<true, true, true> product(ws, rows, d, hidden);
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
  if ((st = AlignedRows::prepare(x, w, cs, flags)) != HPRN_OK) return st;
  Product q;
  q.a = {x.data(), x.ld()};
  q.b = {w.data(), w.ld()};
  q.m = rows, q.n = d, q.depth = hidden, q.pair_offset = d;
  return with_type_and_act(dtype, act, [&](auto t, auto a) {
    using T = decltype(t);
    GatedEpilogue<T, decltype(a)::value> e;
    e.out = Out16(out, out_row_stride, d);
    if (gate_up) {
      e.gate = Out32(gate_up, gate_up_row_stride, d);
      e.up = Out32(gate_up + d, gate_up_row_stride, d);
    }
    return product.launch<T>(q, e, cs, flags, "gated_linear");
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
  const AlignedRows x(ws, input, rows, hidden, input_row_stride, (gate_up ? 0 : 2) * d);
  const AlignedRows w(ws, weight, 2 * d, hidden, weight_row_stride, gate_up ? 0 : rows);
  const int64_t s_ld = round_up(2 * d, 16);
  uint16_t* s = ws.take<uint16_t>(rows * s_ld);
  // Without the kept products the first sums are needed again.
  const PlannedProduct<true, true, true> again(ws, gate_up ? 0 : rows, d, hidden);
  const PlannedProduct<false, true, false> to_input(ws, rows, hidden, 2 * d);
  const PlannedProduct<false, false, false> to_weight(ws, 2 * d, hidden, rows);
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
  if ((st = AlignedRows::prepare(x, w, cs, flags)) != HPRN_OK) return st;
  const char* what = "gated_linear_backward";
  if (rows > 0 && d > 0) {
    st = with_type_and_act(dtype, act, [&](auto t, auto a) {
      using T = decltype(t);
      constexpr int kAct = decltype(a)::value;
      if (gate_up) {
        const GatedGradArgs g{static_cast<const uint16_t*>(grad_out), grad_out_row_stride, gate_up,
                              gate_up_row_stride, s, s_ld, rows, d};
        const bool wide = d % 8 == 0 && tma_rows(grad_out, rows, grad_out_row_stride) &&
                          aligned(gate_up, 16) && (rows <= 1 || gate_up_row_stride % 4 == 0);
        const int64_t ctas = wide ? (rows * (d / 8) + 255) / 256 : rows * ((d + 1023) / 1024);
        const int64_t most = 16 * dev->sm_count;
        const dim3 grid(static_cast<unsigned>(ctas < most ? ctas : most));
        return launch_rows(wide ? gated_grad_vectors<T, kAct> : gated_grad_elements<T, kAct>, grid, dim3(256),
                           cs, flags, what, g);
      }
      Product q;
      q.a = {x.data(), x.ld()};
      q.b = {w.data(), w.ld()};
      q.m = rows, q.n = d, q.depth = hidden, q.pair_offset = d;
      GatedGradEpilogue<T, kAct> e;
      e.dout = static_cast<const uint16_t*>(grad_out), e.dout_ld = grad_out_row_stride;
      e.dout_aligned = tma_rows(grad_out, rows, grad_out_row_stride);
      e.gate = Out16(s, s_ld, d), e.up = Out16(s + d, s_ld, d);
      return again.launch<T>(q, e, cs, flags, what);
    });
    if (st != HPRN_OK) return st;
  }
  // Without rows the weight's gradient is zero, without columns the input's:
  // sums of no terms.
  auto gradients = [&](auto t) {
    using T = decltype(t);
    Product q;
    q.a = {s, s_ld};
    q.b = {w.data(), w.ld()};
    q.m = rows, q.n = hidden, q.depth = 2 * d;
    StoreEpilogue<T> e;
    e.out = Out16(grad_input, grad_input_row_stride, hidden);
    const int r = to_input.launch<T>(q, e, cs, flags, what);
    if (r != HPRN_OK) return r;
    q.b = {x.data(), x.ld()};
    q.m = 2 * d, q.depth = rows;
    e.out = Out16(grad_weight, grad_weight_row_stride, hidden);
    return to_weight.launch<T>(q, e, cs, flags, what);
  };
  return dtype == HPRN_DTYPE_BF16 ? gradients(__nv_bfloat16{}) : gradients(__half{});
}

}  // extern "C"
