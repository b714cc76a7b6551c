// The norms on both sides of a gated block, one pass over a row:
//   y_j = x_j inv_x p_j,  inv_x = rsqrt(mean(x^2) + eps)   (y = x without p)
//   t_j = a r_j + g_j y_j                                  the new residual
//   out_j = t_j inv_t w_j,  inv_t = rsqrt(mean(t^2) + eps)
// x is a block's output, p the weight of the norm after the block, a the scale
// of the residual r, g the gate (absent, one value or one row of values for
// every `rows_per_gate` rows), w the weight of the norm before the next block.
// t stays in fp32 registers between its two uses and is rounded once into the
// residual; out comes from the unrounded t.
//
// Its gradients, D that of out, E that of t from its other uses, n = t inv_t,
// m = x inv_x (m = x and p = 1 without p), means over a row:
//   dt = inv_t (w D - n mean(w D n)) + E
//   dr = a dt,  dg = sum of dt m p over what shares the gate,
//   dx = inv_x (p g dt - m mean(p g dt m)),  dp = sum over rows of g dt m,
//   dw = sum over rows of D n
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <string>

#include "rows.cuh"
#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

struct BlockNormArgs {
  uint16_t* out;
  uint16_t* t;  // the new residual
  const uint16_t* x;
  const uint16_t* r;
  const uint16_t* p;  // or null
  const uint16_t* w;
  const uint16_t* g;  // or null
  int64_t out_stride, t_stride, x_stride, r_stride, g_stride;
  int32_t rows, hidden;
  uint32_t rows_per_gate;
  int32_t gate_row;  // the gate is a row of `hidden` values
  int32_t row_threads, nvec;
  float scale, eps, inv_hidden;
};

// Rows held in registers: a CTA works on blockDim / row_threads rows, each
// thread on VPT vectors of VEC bytes.
template <typename T, int VEC, int VPT>
__global__ void __launch_bounds__(VPT * VEC > 32 ? 512 : 1024) block_norm_rows(BlockNormArgs a) {
  constexpr int P = Pairs<VEC>::kCount;
  __shared__ float part[2][32];
  const int in = threadIdx.x % a.row_threads, group = threadIdx.x / a.row_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / a.row_threads) + group;
  const int warps = a.row_threads / 32, first_warp = group * warps;
  const bool valid = row < a.rows;
  auto inside = [&](int k) { return valid && in + k * a.row_threads < a.nvec; };
  auto at = [&](int k) { return static_cast<int64_t>(in + k * a.row_threads) * Vec<VEC>::kElems; };
  const uint64_t once = policy_evict_first(), keep = policy_evict_last();
  pdl_wait();

  Vec<VEC> x[VPT], r[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (inside(k)) x[k] = ld_stream<VEC>(a.x + row * a.x_stride + at(k), once);
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (inside(k)) r[k] = ld_stream<VEC>(a.r + row * a.r_stride + at(k), once);
  const uint16_t* gate = a.g && valid ? a.g + (static_cast<uint32_t>(row) / a.rows_per_gate) * a.g_stride : nullptr;
  float gate_one = 1.f;
  if (gate && !a.gate_row) gate_one = unpack1<T>(gate[0]);
  float inv_x = 1.f;
  if (a.p) {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (!inside(k)) break;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float2 v = pair_of<T, VEC>(x[k], e);
        s = __ffma2_rn(v, v, s);
      }
    }
    inv_x = rsqrtf(row_sum(s.x + s.y, part[0], warps, first_warp) * a.inv_hidden + a.eps);
  }
  float2 t[VPT][P], s = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (!inside(k)) break;
    Vec<VEC> p, g, o;
    if (a.p) p = ld_weight<VEC>(a.p + at(k), keep);
    if (gate && a.gate_row) g = ld_weight<VEC>(gate + at(k), keep);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      float2 y = pair_of<T, VEC>(x[k], e);
      if (a.p) y = __fmul2_rn(__fmul2_rn(y, make_float2(inv_x, inv_x)), pair_of<T, VEC>(p, e));
      if (gate && a.gate_row) y = __fmul2_rn(y, pair_of<T, VEC>(g, e));
      else y = __fmul2_rn(y, make_float2(gate_one, gate_one));
      t[k][e] = __ffma2_rn(pair_of<T, VEC>(r[k], e), make_float2(a.scale, a.scale), y);
      s = __ffma2_rn(t[k][e], t[k][e], s);
      set_pair<T, VEC>(o, e, t[k][e]);
    }
    st_global<VEC>(a.t + row * a.t_stride + at(k), o);
  }
  const float inv_t = rsqrtf(row_sum(s.x + s.y, part[1], warps, first_warp) * a.inv_hidden + a.eps);
  pdl_trigger();
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (!inside(k)) break;
    const Vec<VEC> w = ld_weight<VEC>(a.w + at(k), keep);
    Vec<VEC> o;
#pragma unroll
    for (int e = 0; e < P; ++e)
      set_pair<T, VEC>(o, e, __fmul2_rn(__fmul2_rn(t[k][e], make_float2(inv_t, inv_t)), pair_of<T, VEC>(w, e)));
    st_global<VEC>(a.out + row * a.out_stride + at(k), o);
  }
}

// Rows too long for registers, one CTA a row, read three times (from L2 after
// the first).  Each thread reads and writes the same elements, and reads x and r
// before it writes them, so out may be x and the residual updated in place.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) block_norm_long_rows(BlockNormArgs a) {
  constexpr int P = Pairs<VEC>::kCount;
  __shared__ float part[2][32];
  const int64_t row = blockIdx.x;
  const int warps = blockDim.x / 32;
  pdl_wait();
  const uint16_t *xr = a.x + row * a.x_stride, *rr = a.r + row * a.r_stride;
  const uint16_t* gate = a.g ? a.g + (static_cast<uint32_t>(row) / a.rows_per_gate) * a.g_stride : nullptr;
  float gate_one = 1.f;
  if (gate && !a.gate_row) gate_one = unpack1<T>(gate[0]);
  float inv_x = 1.f;
  if (a.p) {
    float2 s = make_float2(0.f, 0.f);
    for (int v = threadIdx.x; v < a.nvec; v += blockDim.x) {
      const Vec<VEC> x = ld_l2<VEC>(xr + static_cast<int64_t>(v) * Vec<VEC>::kElems);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float2 q = pair_of<T, VEC>(x, e);
        s = __ffma2_rn(q, q, s);
      }
    }
    inv_x = rsqrtf(row_sum(s.x + s.y, part[0], warps, 0) * a.inv_hidden + a.eps);
  }
  float2 t[P];
  Vec<VEC> rounded;
  auto total = [&](int64_t at) {
    const Vec<VEC> x = ld_l2<VEC>(xr + at), r = ld_l2<VEC>(rr + at);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      float2 y = pair_of<T, VEC>(x, e);
      if (a.p) {
        const float2 p = load_pair<T, VEC>(a.p + at, e);
        y = __fmul2_rn(__fmul2_rn(y, make_float2(inv_x, inv_x)), p);
      }
      if (gate && a.gate_row) y = __fmul2_rn(y, load_pair<T, VEC>(gate + at, e));
      else y = __fmul2_rn(y, make_float2(gate_one, gate_one));
      t[e] = __ffma2_rn(pair_of<T, VEC>(r, e), make_float2(a.scale, a.scale), y);
      set_pair<T, VEC>(rounded, e, t[e]);
    }
  };
  float2 s = make_float2(0.f, 0.f);
  for (int v = threadIdx.x; v < a.nvec; v += blockDim.x) {
    total(static_cast<int64_t>(v) * Vec<VEC>::kElems);
#pragma unroll
    for (int e = 0; e < P; ++e) s = __ffma2_rn(t[e], t[e], s);
  }
  const float inv_t = rsqrtf(row_sum(s.x + s.y, part[1], warps, 0) * a.inv_hidden + a.eps);
  pdl_trigger();
  for (int v = threadIdx.x; v < a.nvec; v += blockDim.x) {
    const int64_t at = static_cast<int64_t>(v) * Vec<VEC>::kElems;
    total(at);
    st_global<VEC>(a.t + row * a.t_stride + at, rounded);
    Vec<VEC> o;
#pragma unroll
    for (int e = 0; e < P; ++e)
      set_pair<T, VEC>(o, e, __fmul2_rn(__fmul2_rn(t[e], make_float2(inv_t, inv_t)), load_pair<T, VEC>(a.w + at, e)));
    st_global<VEC>(a.out + row * a.out_stride + at, o);
  }
}

// ---------------------------------------------------------------------------
// Gradients.

struct BlockGradArgs {
  uint16_t *dx, *dr, *dp, *dw, *dg;  // dp, dg: or null
  const uint16_t *d, *e, *x, *t, *p, *w, *g;  // e, p, g: or null
  int64_t dx_stride, dr_stride, dg_stride, d_stride, e_stride, x_stride, t_stride, g_stride;
  int64_t rows, hidden;
  int64_t rows_per_gate, gates;
  bool gate_row;  // the gate is a row of `hidden` values
  bool gate_each;  // ... of its own for every row
  float scale, eps;
  float4* stats;      // per row: {inv_t, mean(w D n), inv_x, mean(p g dt m)}
  float* gate_sums;   // per row: sum of dt m p, where the gate is one value
  // Sums over the rows of a part (`parts` for each gate where the gate is a
  // shared row, else `parts` in all): of D n, and of dt m where the gate is a
  // shared row, else of g dt m.
  float *dw_parts, *m_parts;
  int64_t parts, part_rows, parts_ld;
};

// The values of one element of row i that the sums and outputs are made of.
template <typename T>
struct BlockGradElement {
  float d, e, n, m, p, g, wd;
  __device__ __forceinline__ BlockGradElement(const BlockGradArgs& a, int64_t i, int64_t j, const uint16_t* gate,
                                         float inv_t, float inv_x) {
    d = unpack1<T>(a.d[i * a.d_stride + j]);
    e = a.e ? unpack1<T>(a.e[i * a.e_stride + j]) : 0.f;
    n = unpack1<T>(a.t[i * a.t_stride + j]) * inv_t;
    m = unpack1<T>(a.x[i * a.x_stride + j]) * inv_x;
    p = a.p ? unpack1<T>(a.p[j]) : 1.f;
    g = gate ? unpack1<T>(gate[a.gate_row ? j : 0]) : 1.f;
    wd = unpack1<T>(a.w[j]) * d;
  }
  __device__ __forceinline__ float dt(float inv_t, float mean) const { return inv_t * (wd - n * mean) + e; }
};

template <typename T>
__device__ __forceinline__ const uint16_t* gate_of(const BlockGradArgs& a, int64_t i) {
  return a.g ? a.g + (static_cast<uint32_t>(i) / static_cast<uint32_t>(a.rows_per_gate)) * a.g_stride : nullptr;
}

// One CTA per row: the row's means.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_stats(BlockGradArgs a) {
  __shared__ float part[4][32];
  pdl_wait();
  const int64_t i = blockIdx.x;
  const uint16_t* gate = gate_of<T>(a, i);
  const float inv_hidden = 1.f / static_cast<float>(a.hidden);
  float st = 0.f, sx = 0.f, sd = 0.f;
  for (int64_t j = threadIdx.x; j < a.hidden; j += 256) {
    const BlockGradElement<T> v(a, i, j, gate, 1.f, 1.f);
    st = fmaf(v.n, v.n, st), sx = fmaf(v.m, v.m, sx), sd = fmaf(v.wd, v.n, sd);
  }
  st = row_sum(st, part[0], 8, 0), sx = row_sum(sx, part[1], 8, 0), sd = row_sum(sd, part[2], 8, 0);
  const float inv_t = rsqrtf(st * inv_hidden + a.eps), inv_x = a.p ? rsqrtf(sx * inv_hidden + a.eps) : 1.f;
  const float mean = sd * inv_t * inv_hidden;
  float s = 0.f;
  for (int64_t j = threadIdx.x; j < a.hidden; j += 256) {
    const BlockGradElement<T> v(a, i, j, gate, inv_t, inv_x);
    s = fmaf(v.dt(inv_t, mean) * v.p * (a.gate_row ? v.g : 1.f), v.m, s);
  }
  s = row_sum(s, part[3], 8, 0);
  if (threadIdx.x != 0) return;
  if (a.gate_sums) a.gate_sums[i] = s;
  if (gate && !a.gate_row) s *= unpack1<T>(gate[0]);
  a.stats[i] = make_float4(inv_t, mean, inv_x, a.p ? s * inv_hidden : 0.f);
}

// A part of the rows x 256 columns per CTA: the rows' outputs, the part's sums.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_columns(BlockGradArgs a) {
  pdl_wait();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (j >= a.hidden) return;
  const bool shared_row = a.gate_row && !a.gate_each;
  const int64_t gates = shared_row ? a.gates : 1, rows = shared_row ? a.rows_per_gate : a.rows;
  for (int64_t part = blockIdx.y; part < gates * a.parts; part += gridDim.y) {
    const int64_t first = part / a.parts * rows, in = part % a.parts * a.part_rows;
    const int64_t end = first + min(rows, in + a.part_rows);
    float sw = 0.f, sm = 0.f;
    for (int64_t i = first + in; i < end; ++i) {
      const float4 st = a.stats[i];
      const BlockGradElement<T> v(a, i, j, gate_of<T>(a, i), st.x, st.z);
      const float dt = v.dt(st.x, st.y);
      a.dr[i * a.dr_stride + j] = pack1<T>(a.scale * dt);
      a.dx[i * a.dx_stride + j] = pack1<T>(a.p ? st.z * (v.p * v.g * dt - v.m * st.w) : v.g * dt);
      sw = fmaf(v.d, v.n, sw);
      sm = fmaf(shared_row ? dt : v.g * dt, v.m, sm);
      if (a.gate_each) a.dg[i * a.dg_stride + j] = pack1<T>(dt * v.m * v.p);
    }
    a.dw_parts[part * a.parts_ld + j] = sw;
    a.m_parts[part * a.parts_ld + j] = sm;
  }
}

// The weights' and a shared gate row's gradients from the parts' sums: 32
// columns a CTA, its 8 warps taking gates (or, where there are none, parts) in
// turn.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_join(BlockGradArgs a) {
  __shared__ float sums[2][8][32];
  pdl_wait();
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  const bool shared_row = a.gate_row && !a.gate_each;
  float sw = 0.f, sp = 0.f;
  if (j < a.hidden) {
    if (shared_row) {
      const float p = a.p ? unpack1<T>(a.p[j]) : 1.f;
      for (int64_t k = ty; k < a.gates; k += 8) {
        float sm = 0.f;
        for (int64_t part = k * a.parts; part < (k + 1) * a.parts; ++part) {
          sw += a.dw_parts[part * a.parts_ld + j];
          sm += a.m_parts[part * a.parts_ld + j];
        }
        sp = fmaf(unpack1<T>(a.g[k * a.g_stride + j]), sm, sp);
        a.dg[k * a.dg_stride + j] = pack1<T>(sm * p);
      }
    } else {
      for (int64_t part = ty; part < a.parts; part += 8) {
        sw += a.dw_parts[part * a.parts_ld + j];
        sp += a.m_parts[part * a.parts_ld + j];
      }
    }
  }
  sums[0][ty][tx] = sw, sums[1][ty][tx] = sp;
  __syncthreads();
  if (ty > 0 || j >= a.hidden) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sw += sums[0][k][tx], sp += sums[1][k][tx];
  a.dw[j] = pack1<T>(sw);
  if (a.dp) a.dp[j] = pack1<T>(sp);
}

// The gradients of gates of one value: one CTA adds up the rows that share one.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_gates(BlockGradArgs a) {
  __shared__ float part[32];
  pdl_wait();
  for (int64_t k = blockIdx.x; k < a.gates; k += gridDim.x) {
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.rows_per_gate; i += 256) s += a.gate_sums[k * a.rows_per_gate + i];
    s = row_sum(s, part, 8, 0);
    if (threadIdx.x == 0) a.dg[k * a.dg_stride] = pack1<T>(s);
    __syncthreads();
  }
}

namespace {

int check_sizes(int64_t rows, int64_t hidden, int64_t rows_per_gate, int64_t gate_width, bool gate, int dtype) {
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (rows < 0 || hidden < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || hidden > kMaxExtent)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows and hidden must be at most 2^30");
  if (gate && (rows_per_gate < 1 || rows % rows_per_gate != 0))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows must be a multiple of rows_per_gate");
  if (gate && gate_width != 1 && gate_width != hidden)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "gate_width must be 1 or hidden");
  return HPRN_OK;
}

// The widest vectors that every row of every tensor is made of.
int vector_bytes(int64_t hidden, std::initializer_list<const void*> rows, std::initializer_list<int64_t> strides) {
  for (int vec : {32, 16, 4}) {
    bool fits = hidden * 2 % vec == 0;
    for (const void* p : rows) fits = fits && aligned(p, vec);
    for (int64_t s : strides) fits = fits && s * 2 % vec == 0;
    if (fits) return vec;
  }
  return 2;
}

using RowsKernel = void (*)(BlockNormArgs);

template <typename T>
RowsKernel rows_kernel(int vec, int vpt) {
  switch (vec * 100 + vpt) {
    case 3201: return block_norm_rows<T, 32, 1>;
    case 3202: return block_norm_rows<T, 32, 2>;
    case 1601: return block_norm_rows<T, 16, 1>;
    case 1602: return block_norm_rows<T, 16, 2>;
    case 401: return block_norm_rows<T, 4, 1>;
    case 402: return block_norm_rows<T, 4, 2>;
    case 404: return block_norm_rows<T, 4, 4>;
    case 408: return block_norm_rows<T, 4, 8>;
    case 201: return block_norm_rows<T, 2, 1>;
    case 202: return block_norm_rows<T, 2, 2>;
    case 204: return block_norm_rows<T, 2, 4>;
    case 208: return block_norm_rows<T, 2, 8>;
    case 216: return block_norm_rows<T, 2, 16>;
    default: return nullptr;
  }
}

template <typename T>
int launch_forward(BlockNormArgs& a, int vec, cudaStream_t stream, unsigned flags) {
  const char* what = "gated_add_rms_norm";
  a.nvec = static_cast<int32_t>(static_cast<int64_t>(a.hidden) * 2 / vec);
  for (int vpt = 1; vpt <= 16; vpt *= 2) {
    const RowsKernel fn = rows_kernel<T>(vec, vpt);
    const int64_t threads = round_up((a.nvec + vpt - 1) / vpt, 32);
    // More vectors a thread leave registers for 512 threads only.
    if (!fn || threads > (vpt * vec > 32 ? 512 : 1024)) continue;
    a.row_threads = static_cast<int32_t>(threads);
    const int groups = threads <= 64 ? static_cast<int>(128 / threads) : 1;
    return launch_rows(fn, dim3(static_cast<unsigned>((a.rows + groups - 1) / groups)),
                       dim3(static_cast<unsigned>(threads * groups)), stream, flags, what, a);
  }
  a.row_threads = 1024;
  if (vec >= 16) {
    a.nvec = static_cast<int32_t>(a.hidden / 8);
    return launch_rows(block_norm_long_rows<T, 16>, dim3(a.rows), dim3(1024), stream, flags, what, a);
  }
  a.nvec = a.hidden;
  return launch_rows(block_norm_long_rows<T, 2>, dim3(a.rows), dim3(1024), stream, flags, what, a);
}

template <typename T>
int launch_backward(const BlockGradArgs& a, cudaStream_t stream, unsigned flags) {
  const char* what = "gated_add_rms_norm_backward";
  int st = HPRN_OK;
  if (a.rows > 0) {
    st = launch_rows(block_grad_stats<T>, dim3(static_cast<unsigned>(a.rows)), dim3(256), stream, flags, what, a);
    if (st != HPRN_OK) return st;
    const int64_t parts = (a.gate_row && !a.gate_each ? a.gates : 1) * a.parts;
    st = launch_rows(block_grad_columns<T>,
                     dim3(static_cast<unsigned>((a.hidden + 255) / 256), static_cast<unsigned>(parts < 65535 ? parts : 65535)),
                     dim3(256), stream, flags, what, a);
    if (st != HPRN_OK) return st;
    if (a.gate_sums) {
      st = launch_rows(block_grad_gates<T>, dim3(static_cast<unsigned>(a.gates < 65535 ? a.gates : 65535)), dim3(256),
                       stream, flags, what, a);
      if (st != HPRN_OK) return st;
    }
  }
  return launch_rows(block_grad_join<T>, dim3(static_cast<unsigned>((a.hidden + 31) / 32)), dim3(256), stream, flags,
                     what, a);
}

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_gated_add_rms_norm(void* out, void* residual_out, const void* input, const void* residual,
                            const void* post_weight, const void* weight, const void* gate, int64_t rows,
                            int64_t hidden, int64_t rows_per_gate, int64_t gate_width, int64_t out_row_stride,
                            int64_t residual_out_row_stride, int64_t input_row_stride, int64_t residual_row_stride,
                            int64_t gate_row_stride, double residual_scale, double eps, int dtype, void* stream,
                            unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL)) return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  int st = check_sizes(rows, hidden, rows_per_gate, gate_width, gate != nullptr, dtype);
  if (st != HPRN_OK) return st;
  const int64_t gates = gate ? rows / rows_per_gate : 1;
  if ((rows > 1 && (out_row_stride < hidden || residual_out_row_stride < hidden || input_row_stride < hidden ||
                    residual_row_stride < hidden)) ||
      (gates > 1 && gate_row_stride < gate_width))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  if (rows == 0 || hidden == 0) return ok();
  if (!out || !residual_out || !input || !residual || !weight)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  for (const void* p : {static_cast<const void*>(out), static_cast<const void*>(residual_out), input, residual,
                        post_weight, weight, gate})
    if (!aligned(p, 2)) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  if (rows == 1) out_row_stride = residual_out_row_stride = input_row_stride = residual_row_stride = hidden;
  if (gates == 1) gate_row_stride = gate_width;
  // The input and the residual may be written in place, each by its own output.
  const bool same_x = out == input && out_row_stride == input_row_stride;
  const bool same_r = residual_out == residual && residual_out_row_stride == residual_row_stride;
  const Extent x = extent16(input, rows, hidden, input_row_stride),
               r = extent16(residual, rows, hidden, residual_row_stride),
               o = extent16(out, rows, hidden, out_row_stride),
               t = extent16(residual_out, rows, hidden, residual_out_row_stride);
  const Extent outs[] = {o, t};
  const Extent ins[] = {extent16(post_weight, 1, hidden, hidden), extent16(weight, 1, hidden, hidden),
                        extent16(gate, gates, gate_width, gate_row_stride)};
  if (!disjoint(outs, ins) || extents_overlap(o, r) || extents_overlap(t, x) || (!same_x && extents_overlap(o, x)) ||
      (!same_r && extents_overlap(t, r)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors, but for out == input and "
                                           "residual_out == residual");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  BlockNormArgs a{};
  a.out = static_cast<uint16_t*>(out), a.t = static_cast<uint16_t*>(residual_out);
  a.x = static_cast<const uint16_t*>(input), a.r = static_cast<const uint16_t*>(residual);
  a.p = static_cast<const uint16_t*>(post_weight), a.w = static_cast<const uint16_t*>(weight);
  a.g = static_cast<const uint16_t*>(gate);
  a.out_stride = out_row_stride, a.t_stride = residual_out_row_stride, a.x_stride = input_row_stride;
  a.r_stride = residual_row_stride, a.g_stride = gate_row_stride;
  a.rows = static_cast<int32_t>(rows), a.hidden = static_cast<int32_t>(hidden);
  a.rows_per_gate = static_cast<uint32_t>(gate ? rows_per_gate : 1);
  a.gate_row = gate && gate_width == hidden;
  a.scale = static_cast<float>(residual_scale), a.eps = static_cast<float>(eps);
  a.inv_hidden = 1.f / static_cast<float>(hidden);
  const bool gate_rows = a.gate_row;
  const int vec = vector_bytes(hidden, {out, residual_out, input, residual, post_weight, weight, gate_rows ? gate : nullptr},
                               {rows > 1 ? out_row_stride : 0, rows > 1 ? residual_out_row_stride : 0,
                                rows > 1 ? input_row_stride : 0, rows > 1 ? residual_row_stride : 0,
                                gate_rows && gates > 1 ? gate_row_stride : 0});
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == HPRN_DTYPE_BF16 ? launch_forward<__nv_bfloat16>(a, vec, cs, flags)
                                  : launch_forward<__half>(a, vec, cs, flags);
}

int hprn_gated_add_rms_norm_backward(
    void* grad_input, void* grad_residual, void* grad_post_weight, void* grad_weight, void* grad_gate,
    const void* grad_out, const void* grad_residual_out, const void* input, const void* residual_out,
    const void* post_weight, const void* weight, const void* gate, int64_t rows, int64_t hidden,
    int64_t rows_per_gate, int64_t gate_width, int64_t grad_input_row_stride, int64_t grad_residual_row_stride,
    int64_t grad_gate_row_stride, int64_t grad_out_row_stride, int64_t grad_residual_out_row_stride,
    int64_t input_row_stride, int64_t residual_out_row_stride, int64_t gate_row_stride, double residual_scale,
    double eps, int dtype, void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  int st = check_sizes(rows, hidden, rows_per_gate, gate_width, gate != nullptr, dtype);
  if (st != HPRN_OK) return st;
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  const int64_t gates = gate ? rows / rows_per_gate : 1;
  if ((rows > 1 && (grad_input_row_stride < hidden || grad_residual_row_stride < hidden ||
                    grad_out_row_stride < hidden || (grad_residual_out && grad_residual_out_row_stride < hidden) ||
                    input_row_stride < hidden || residual_out_row_stride < hidden)) ||
      (gate && gates > 1 && (gate_row_stride < gate_width || grad_gate_row_stride < gate_width)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  BlockGradArgs a{};
  a.dx = static_cast<uint16_t*>(grad_input), a.dr = static_cast<uint16_t*>(grad_residual);
  a.dp = static_cast<uint16_t*>(grad_post_weight), a.dw = static_cast<uint16_t*>(grad_weight);
  a.dg = static_cast<uint16_t*>(grad_gate);
  a.d = static_cast<const uint16_t*>(grad_out), a.e = static_cast<const uint16_t*>(grad_residual_out);
  a.x = static_cast<const uint16_t*>(input), a.t = static_cast<const uint16_t*>(residual_out);
  a.p = static_cast<const uint16_t*>(post_weight), a.w = static_cast<const uint16_t*>(weight);
  a.g = static_cast<const uint16_t*>(gate);
  a.dx_stride = grad_input_row_stride, a.dr_stride = grad_residual_row_stride, a.dg_stride = grad_gate_row_stride;
  a.d_stride = grad_out_row_stride, a.e_stride = grad_residual_out_row_stride, a.x_stride = input_row_stride;
  a.t_stride = residual_out_row_stride, a.g_stride = gate_row_stride;
  a.rows = rows, a.hidden = hidden;
  a.rows_per_gate = gate ? rows_per_gate : 1, a.gates = gates;
  // (With hidden 1 a gate of one value is a row of one.)
  a.gate_row = gate && gate_width == hidden, a.gate_each = a.gate_row && rows_per_gate == 1;
  a.scale = static_cast<float>(residual_scale), a.eps = static_cast<float>(eps);
  const bool shared_row = a.gate_row && !a.gate_each;
  const int64_t share = shared_row ? rows_per_gate : rows;
  a.parts = shared_row ? (64 + gates - 1) / (gates > 0 ? gates : 1) : 64;
  if (a.parts > share) a.parts = share > 0 ? share : 1;
  a.part_rows = (share + a.parts - 1) / a.parts;
  a.parts = a.part_rows > 0 ? (share + a.part_rows - 1) / a.part_rows : 0;
  Workspace ws(workspace, *workspace_bytes);
  a.stats = ws.take<float4>(rows);
  a.gate_sums = ws.take<float>(gate && !a.gate_row ? rows : 0);
  if (!gate || a.gate_row) a.gate_sums = nullptr;
  a.parts_ld = round_up(hidden, 8);
  a.dw_parts = ws.take<float>((shared_row ? gates : 1) * a.parts * a.parts_ld);
  a.m_parts = ws.take<float>((shared_row ? gates : 1) * a.parts * a.parts_ld);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if (!grad_weight || !weight || (post_weight && !grad_post_weight) ||
      (rows > 0 && (!grad_input || !grad_residual || !grad_out || !input || !residual_out || (gate && !grad_gate))))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!post_weight) a.dp = nullptr;
  for (const void* p : {static_cast<const void*>(grad_input), static_cast<const void*>(grad_residual),
                        static_cast<const void*>(grad_post_weight), static_cast<const void*>(grad_weight),
                        static_cast<const void*>(grad_gate), grad_out, grad_residual_out, input, residual_out,
                        post_weight, weight, gate})
    if (!aligned(p, 2)) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                         extent16(grad_residual, rows, hidden, grad_residual_row_stride),
                         extent16(a.dp, 1, hidden, hidden), extent16(grad_weight, 1, hidden, hidden),
                         extent16(gate ? grad_gate : nullptr, gates, gate_width, grad_gate_row_stride)};
  const Extent ins[] = {extent16(grad_out, rows, hidden, grad_out_row_stride),
                        extent16(grad_residual_out, rows, hidden, grad_residual_out_row_stride),
                        extent16(input, rows, hidden, input_row_stride),
                        extent16(residual_out, rows, hidden, residual_out_row_stride),
                        extent16(post_weight, 1, hidden, hidden), extent16(weight, 1, hidden, hidden),
                        extent16(gate, gates, gate_width, gate_row_stride)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == HPRN_DTYPE_BF16 ? launch_backward<__nv_bfloat16>(a, cs, flags)
                                  : launch_backward<__half>(a, cs, flags);
}

}  // extern "C"
