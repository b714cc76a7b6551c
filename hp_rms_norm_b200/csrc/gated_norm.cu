// The norms on both sides of a gated block, one pass over a row:
//   y_j = x_j inv_x p_j,  inv_x = rsqrt(mean(x^2) + eps)   (y = x without p)
//   t_j = a r_j + g_j y_j                                  the new residual
//   out_j = t_j inv_t w_j,  inv_t = rsqrt(mean(t^2) + eps)
// x is a block's output, p the weight of the norm after the block, a the scale
// of the residual r, g the gate (absent, one value or one row of values for
// every `rows_per_gate` rows), w the weight of the norm before the next block.
// t stays in fp32 registers between its two uses and is rounded once into the
// residual; out comes from the unrounded t.
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <string>

#include "gated_norm.cuh"
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
  // Rows that are worked on at once where the grid is larger than that, else 0.
  int32_t wave_rows;
  float scale, eps, inv_hidden;
};

// Rows held in registers: a CTA works on blockDim / row_threads rows, each
// thread on VPT vectors of VEC bytes.  kLoose: rows that start anywhere (rows.cuh).
// kGateRow: the gate is a row of values; else one value, or none.  kMost: the threads
// of a CTA at most, two of which share an SM where they are fewer than 1024.
template <typename T, int VEC, int VPT, bool kLoose, bool kPost, bool kGateRow, int kMost = 1024>
__global__ void __launch_bounds__(kMost, kMost < 1024 ? 2 : 1) block_norm_rows(BlockNormArgs a) {
  static_assert(!kLoose || VEC == 16, "loose rows are read in vectors of eight elements");
  constexpr int P = VEC / 4;
  __shared__ float part[2][32];
  const int in = threadIdx.x % a.row_threads, group = threadIdx.x / a.row_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / a.row_threads) + group;
  const int warps = a.row_threads / 32, first_warp = group * warps;
  const bool valid = row < a.rows;
  // (Of a loose row, what a warp has some of: its lanes store together.)
  const int from = kLoose ? in & ~31 : in;
  auto inside = [&](int k) { return valid && from + k * a.row_threads < a.nvec; };
  auto vector = [&](int k) { return in + k * a.row_threads; };
  const uint64_t once = policy_evict_first(), keep = policy_evict_last();
  auto load = [&](const uint16_t* base, int64_t stride, int k) {
    Vec<VEC> v;
    if constexpr (kLoose) load_loose(v.w, loose_row(base, row, a.rows, stride, a.hidden), vector(k));
    else v = ld_stream<VEC>(base + row * stride + vector(k) * Vec<VEC>::kElems, once);
    return v;
  };
  auto weight = [&](const uint16_t* p, int k) {
    Vec<VEC> v;
    if constexpr (kLoose) load_loose(v.w, LooseRow{p, a.hidden, false, false}, vector(k));
    else v = ld_weight<VEC>(p + vector(k) * Vec<VEC>::kElems, keep);
    return v;
  };
  auto store = [&](uint16_t* base, int64_t stride, int k, const Vec<VEC>& v) {
    if constexpr (kLoose) store_loose(base + row * stride, a.hidden, vector(k), v.w);
    else st_global<VEC>(base + row * stride + vector(k) * Vec<VEC>::kElems, v);
  };
  // The first rows into L2 while the preceding grid drains, and then the row that
  // will take this one's place.
  auto ahead = [&](int64_t i) {
    if (in != 0 || i >= a.rows) return;
    prefetch_l2(a.x + i * a.x_stride, static_cast<uint64_t>(a.hidden) * 2);
    prefetch_l2(a.r + i * a.r_stride, static_cast<uint64_t>(a.hidden) * 2);
  };
  if (a.wave_rows == 0 || row < a.wave_rows) ahead(row);
  pdl_wait();

  Vec<VEC> x[VPT], r[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (inside(k)) x[k] = load(a.x, a.x_stride, k);
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (inside(k)) r[k] = load(a.r, a.r_stride, k);
  if (a.wave_rows > 0) {
    ahead(row + a.wave_rows);
    pdl_trigger();
  }
  const uint16_t* gate = a.g && valid ? a.g + (static_cast<uint32_t>(row) / a.rows_per_gate) * a.g_stride : nullptr;
  float inv_x = 1.f;
  if constexpr (kPost) {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (!inside(k)) break;
#pragma unroll
      for (int e = 0; e < P; ++e) s = fma_pair<T>(x[k].w[e], x[k].w[e], s);
    }
    inv_x = rsqrtf(row_sum(s.x + s.y, part[0], warps, first_warp) * a.inv_hidden + a.eps);
  }
  if constexpr (!kGateRow) {
    if (gate) inv_x *= unpack1<T>(gate[0]);
  }
  const float2 by = make_float2(inv_x, inv_x), scale = make_float2(a.scale, a.scale);
  float2 t[VPT][P], s = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (!inside(k)) break;
    Vec<VEC> p, g, o;
    if constexpr (kPost) p = weight(a.p, k);
    if constexpr (kGateRow) g = weight(gate, k);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      float2 y = __fmul2_rn(unpack2<T>(x[k].w[e]), by);
      if constexpr (kPost && kGateRow) y = __fmul2_rn(y, mul_pair<T>(p.w[e], g.w[e]));
      else if constexpr (kPost) y = __fmul2_rn(y, unpack2<T>(p.w[e]));
      else if constexpr (kGateRow) y = __fmul2_rn(y, unpack2<T>(g.w[e]));
      t[k][e] = __ffma2_rn(unpack2<T>(r[k].w[e]), scale, y);
      s = __ffma2_rn(t[k][e], t[k][e], s);
      o.w[e] = pack2<T>(t[k][e].x, t[k][e].y);
    }
    store(a.t, a.t_stride, k, o);
  }
  const float inv_t = rsqrtf(row_sum(s.x + s.y, part[1], warps, first_warp) * a.inv_hidden + a.eps);
  if (a.wave_rows == 0) pdl_trigger();
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (!inside(k)) break;
    const Vec<VEC> w = weight(a.w, k);
    Vec<VEC> o;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      const float2 y = __fmul2_rn(__fmul2_rn(t[k][e], make_float2(inv_t, inv_t)), unpack2<T>(w.w[e]));
      o.w[e] = pack2<T>(y.x, y.y);
    }
    store(a.out, a.out_stride, k, o);
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

namespace {

// The widest vectors that every row of every tensor is made of: 32 or 16 bytes, or 0.
int vector_bytes(int64_t hidden, std::initializer_list<const void*> rows, std::initializer_list<int64_t> strides) {
  for (int vec : {32, 16}) {
    bool fits = hidden * 2 % vec == 0;
    for (const void* p : rows) fits = fits && aligned(p, vec);
    for (int64_t s : strides) fits = fits && s * 2 % vec == 0;
    if (fits) return vec;
  }
  return 0;
}

using RowsKernel = void (*)(BlockNormArgs);

template <typename T, bool kPost, bool kGateRow>
RowsKernel rows_kernel(int vec, int vpt, int64_t threads) {
  // The sums of a row leave an SM idle meanwhile unless it has a second CTA: in the
  // 48 or 40 registers that 640 or 768 threads have then (4096 x 10240 72.7 us with one,
  // 52.2 with two; x 12288 83.4 and 65.2, for all of 24 bytes spilled).
  if (vec == 32 && vpt == 1 && threads > 512 && threads <= 768)
    return threads <= 640 ? block_norm_rows<T, 32, 1, false, kPost, kGateRow, 640>
                          : block_norm_rows<T, 32, 1, false, kPost, kGateRow, 768>;
  if (vec == 32) return vpt == 1 ? block_norm_rows<T, 32, 1, false, kPost, kGateRow> : nullptr;
  if (vec == 16) return vpt == 1 ? block_norm_rows<T, 16, 1, false, kPost, kGateRow> : block_norm_rows<T, 16, 2, false, kPost, kGateRow>;
  return vpt == 1 ? block_norm_rows<T, 16, 1, true, kPost, kGateRow> : block_norm_rows<T, 16, 2, true, kPost, kGateRow>;
}

template <typename T>
int launch_forward(BlockNormArgs& a, int vec, const DeviceInfo* dev, cudaStream_t stream, unsigned flags) {
  const char* what = "gated_add_rms_norm";
  const int64_t elems = vec > 0 ? vec / 2 : 8;
  a.nvec = static_cast<int32_t>((a.hidden + elems - 1) / elems);
  for (int vpt = 1; vpt <= 2; ++vpt) {
    const int64_t threads = round_up((a.nvec + vpt - 1) / vpt, 32);
    const RowsKernel fn = a.p ? (a.gate_row ? rows_kernel<T, true, true>(vec, vpt, threads) : rows_kernel<T, true, false>(vec, vpt, threads))
                              : (a.gate_row ? rows_kernel<T, false, true>(vec, vpt, threads) : rows_kernel<T, false, false>(vec, vpt, threads));
    if (!fn || threads > 1024) continue;
    a.row_threads = static_cast<int32_t>(threads);
    const int groups = threads <= 64 ? static_cast<int>(128 / threads) : 1;
    const int64_t wave = first_wave_ctas(dev, reinterpret_cast<const void*>(fn), static_cast<int>(threads) * groups) * groups;
    // Rows that start anywhere are bound by issue: many of them by two vectors a thread,
    // half the sums over threads for each (us, one / two): 3084 x 2001 22.6 / 20.1, x 5001
    // 55 / 48; of fewer waves 592 x 2001 5.4 / 6.5, x 5001 11.3 / 12.5; where that leaves more
    // threads idle, 3084 x 515 8.9 / 10.7.
    if (vec == 0 && vpt == 1 && wave > 0 && a.rows > 4 * wave && 2 * round_up((a.nvec + 1) / 2, 32) <= threads) continue;
    a.wave_rows = wave > 0 && a.rows > wave ? static_cast<int32_t>(wave) : 0;
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
  int st = check_block_norm(rows, hidden, rows_per_gate, gate_width, gate != nullptr, dtype);
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
  return dtype == HPRN_DTYPE_BF16 ? launch_forward<__nv_bfloat16>(a, vec, dev, cs, flags)
                                  : launch_forward<__half>(a, vec, dev, cs, flags);
}

int hprn_test_loose_reads(int64_t rows, int64_t hidden, int64_t row_stride, int64_t start, int64_t* out) {
  using namespace hprn;
  if (rows < 1 || hidden < 1 || rows > 4096 || hidden > 65536 || row_stride < hidden || row_stride > 65536 || start < 0 ||
      start > 7 || !out)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows, hidden, strides and starts of a small tensor");
  // (Only addresses: nothing is read.)
  const uint16_t* base = reinterpret_cast<const uint16_t*>(uintptr_t{1} << 30) + start;
  const int n = static_cast<int>(hidden), lanes = (n + 255) / 256 * 32;
  const int64_t end = (rows - 1) * row_stride + hidden;
  out[0] = out[1] = out[2] = 0;
  for (int64_t i = 0; i < rows; ++i) {
    const LooseRow r = loose_row(base, i, rows, row_stride, n);
    const int o = granule_offset(r.p);
    for (int v = 0; v < lanes; ++v) {
      int64_t from = 8 * v, to = from + 8 < hidden ? from + 8 : hidden;  // of the row
      if (reads_granule(r, o, v)) from -= o, to = from + (reads_next(r, o, v) ? 16 : 8);
      if (to > from) {
        const int64_t before = -(i * row_stride + from), behind = i * row_stride + to - end;
        if (before > out[0]) out[0] = before;
        if (behind > out[1]) out[1] = behind;
      }
      // Elements of the row that the vector has and that were not read.
      const int64_t last = 8 * v + 8 < hidden ? 8 * v + 8 : hidden;
      if (8 * v < last && (to < last || from > 8 * v)) ++out[2];
    }
  }
  return ok();
}

}  // extern "C"
