// Linear layers in 8-bit integers: tokens quantised with one scale each (by
// themselves, or as the output of an RMSNorm), the weight with one scale for
// each output channel.
//   scale_i = max(max_j |y_ij|, 1e-12) / 127,  q_ij = round(y_ij (1 / scale_i))
//   out_ij = (sum_k q_ik v_jk) scale_i channel_j + bias_j
// The sum is an exact 32-bit integer from the tensor cores; it is rounded to
// fp32 once, and the result to 16 bits once.
//   Of a norm y_ij = (t_ij w_j) inv_i: its largest is known before inv is.  That order
// and 1 / scale in place of a division each cost y / scale one fp32 rounding, at most
// 127 2^-24 of a step: a code within 2^-16 of a tie may be its neighbour, half a step off
// like the other one.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "few_rows.cuh"
#include "matmul.cuh"
#include "rows.cuh"
#include "runtime.cuh"

namespace hprn {

// ---------------------------------------------------------------------------
// Quantised rows: y = RMSNorm(t) w with t = x [+ r], or y = x without a weight.

// (quantize_int8, nothing in L2: 4096 x 4096 9.9 us, x 8192 19.8, 0.78 of the copy rate;
// x 16384 54.3, one row of 1024 threads an SM; 3084 x 1001 5.6; one row 1.4.)
struct QuantArgs {
  int8_t* q;
  float* scales;
  uint16_t* t;        // the sum x + r, where there is an r
  const uint16_t* x;
  const uint16_t* r;  // or null
  const uint16_t* w;  // or null: no norm
  int64_t q_stride, t_stride, x_stride, r_stride;
  int32_t rows, hidden;
  int32_t row_threads, nvec;
  int32_t wave_rows;  // as in gated_norm.cu
  float eps, inv_hidden;
};

// max(m, |a|, |b|), NaN where one is: a row with a NaN gets a NaN scale.
__device__ __forceinline__ float amax_nan(float m, float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return d;
}

// The largest over the threads that hold a row, as row_sum.
__device__ __forceinline__ float row_amax(float v, float* part, int warps, int first_warp) {
  auto over = [](float m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = amax_nan(m, __shfl_xor_sync(~0u, m, o), 0.f);
    return m;
  };
  v = over(v);
  if (warps == 1) return v;
  const int lane = threadIdx.x % 32;
  if (lane == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  return over(lane < warps ? part[first_warp + lane] : 0.f);
}

// A pair's codes, the first in the low byte.  (cvt.rni of a NaN is 0.)
__device__ __forceinline__ uint32_t codes_of(float2 y, float inv) {
  uint32_t d;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(d) : "r"(__float2int_rn(y.y * inv)), "r"(__float2int_rn(y.x * inv)));
  return d & 0xffffu;
}

template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* q, const float2 (&y)[Pairs<VEC>::kCount], float inv) {
  if constexpr (VEC == 2) {
    *q = static_cast<int8_t>(codes_of(y[0], inv));
  } else {
    Vec<VEC / 2> o;
#pragma unroll
    for (int k = 0; k < VEC / 8; ++k) o.w[k] = codes_of(y[2 * k], inv) | codes_of(y[2 * k + 1], inv) << 16;
    st_global<VEC / 2>(q, o);
  }
}

// Codes 8 v to 8 v + 7 of a row of n bytes that starts anywhere, v neighbouring in
// neighbouring lanes: whole words of eight inside a warp's span, as store_loose.
__device__ __forceinline__ void store_codes_loose(int8_t* row, int n, int v, const float2 (&y)[4], float inv) {
  const int o = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 7), lane = threadIdx.x % 32;
  const LooseEdge edge = loose_edge(n, v, o);
  const uint64_t lo = codes_of(y[0], inv) | codes_of(y[1], inv) << 16, hi = codes_of(y[2], inv) | codes_of(y[3], inv) << 16;
  const uint64_t own = lo | hi << 32, before = __shfl_up_sync(~0u, own, 1);
  const uint64_t over = __shfl_sync(~0u, own, edge.lane);
  if (edge.mine) row[edge.unit] = static_cast<int8_t>(over >> (8 * edge.at));
  if ((lane > 0 || o == 0) && 8 * v - o + 8 <= n)
    *reinterpret_cast<uint64_t*>(row + 8 * v - o) = o > 0 ? before >> (64 - 8 * o) | own << (8 * o) : own;
}

// Rows held in registers, laid out over threads as in gated_norm.cu.
template <typename T, int VEC, int VPT, bool kLoose, bool kNorm, int kMost = 1024>
__global__ void __launch_bounds__(kMost, kMost < 1024 ? 2 : 1) quant_rows(QuantArgs a) {
  static_assert(!kLoose || VEC == 16, "loose rows are read in vectors of eight elements");
  constexpr int P = VEC / 4;
  __shared__ float part[2][32];
  const int in = threadIdx.x % a.row_threads, group = threadIdx.x / a.row_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / a.row_threads) + group;
  const int warps = a.row_threads / 32, first_warp = group * warps;
  const bool valid = row < a.rows;
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
  auto ahead = [&](int64_t i) {
    if (in != 0 || i >= a.rows) return;
    prefetch_l2(a.x + i * a.x_stride, static_cast<uint64_t>(a.hidden) * 2);
    if (a.r) prefetch_l2(a.r + i * a.r_stride, static_cast<uint64_t>(a.hidden) * 2);
  };
  if (a.wave_rows == 0 || row < a.wave_rows) ahead(row);
  pdl_wait();

  Vec<VEC> x[VPT], r[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (inside(k)) x[k] = load(a.x, a.x_stride, k);
  if (a.r) {
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (inside(k)) r[k] = load(a.r, a.r_stride, k);
  }
  if (a.wave_rows > 0) {
    ahead(row + a.wave_rows);
    pdl_trigger();
  }
  float2 y[VPT][P], s = make_float2(0.f, 0.f);
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (!inside(k)) break;
    Vec<VEC> w;
    if constexpr (kNorm) {
      if constexpr (kLoose) load_loose(w.w, LooseRow{a.w, a.hidden, false, false}, vector(k));
      else w = ld_weight<VEC>(a.w + vector(k) * Vec<VEC>::kElems, keep);
    }
    if (a.r) {
      Vec<VEC> o;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        y[k][e] = __fadd2_rn(unpack2<T>(x[k].w[e]), unpack2<T>(r[k].w[e]));
        o.w[e] = pack2<T>(y[k][e].x, y[k][e].y);
      }
      if constexpr (kLoose) store_loose(a.t + row * a.t_stride, a.hidden, vector(k), o.w);
      else st_global<VEC>(a.t + row * a.t_stride + vector(k) * Vec<VEC>::kElems, o);
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) y[k][e] = unpack2<T>(x[k].w[e]);
    }
#pragma unroll
    for (int e = 0; e < P; ++e) {
      if constexpr (kNorm) {
        s = __ffma2_rn(y[k][e], y[k][e], s);
        y[k][e] = __fmul2_rn(y[k][e], unpack2<T>(w.w[e]));
      }
      most = amax_nan(most, y[k][e].x, y[k][e].y);
    }
  }
  float inv = 1.f;
  if constexpr (kNorm) inv = rsqrtf(row_sum(s.x + s.y, part[0], warps, first_warp) * a.inv_hidden + a.eps);
  // max |y inv| = max |y| inv, rounded once: rounding keeps the order.
  most = row_amax(most, part[1], warps, first_warp) * inv;
  if (a.wave_rows == 0) pdl_trigger();
  const float scale = amax_nan(1e-12f, most, 0.f) / 127.f, by = 1.f / scale;
  if (valid && in == 0) a.scales[row] = scale;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (!inside(k)) break;
    if constexpr (kNorm) {
#pragma unroll
      for (int e = 0; e < P; ++e) y[k][e] = __fmul2_rn(y[k][e], make_float2(inv, inv));
    }
    int8_t* q = a.q + row * a.q_stride;
    if constexpr (kLoose) store_codes_loose(q, a.hidden, vector(k), y[k], by);
    else store_codes<VEC>(q + vector(k) * Vec<VEC>::kElems, y[k], by);
  }
}

// Rows too long for registers, one CTA a row, read twice.  The second reading
// finds the same x and r: where the residual is updated in place, its new value
// is written then.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) quant_long_rows(QuantArgs a) {
  constexpr int P = Pairs<VEC>::kCount;
  __shared__ float part[2][32];
  const int64_t row = blockIdx.x;
  pdl_wait();
  Vec<VEC> rounded;
  float2 y[P], sum[P];
  auto load = [&](int64_t at) {
    const Vec<VEC> x = ld_l2<VEC>(a.x + row * a.x_stride + at);
    Vec<VEC> r;
    if (a.r) r = ld_l2<VEC>(a.r + row * a.r_stride + at);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      sum[e] = pair_of<T, VEC>(x, e);
      if (a.r) {
        sum[e] = __fadd2_rn(sum[e], pair_of<T, VEC>(r, e));
        set_pair<T, VEC>(rounded, e, sum[e]);
      }
      y[e] = a.w ? __fmul2_rn(sum[e], load_pair<T, VEC>(a.w + at, e)) : sum[e];
    }
  };
  float2 s = make_float2(0.f, 0.f);
  float most = 0.f;
  for (int v = threadIdx.x; v < a.nvec; v += 1024) {
    load(static_cast<int64_t>(v) * Vec<VEC>::kElems);
#pragma unroll
    for (int e = 0; e < P; ++e) s = __ffma2_rn(sum[e], sum[e], s), most = amax_nan(most, y[e].x, y[e].y);
  }
  float inv = 1.f;
  if (a.w) inv = rsqrtf(row_sum(s.x + s.y, part[0], 32, 0) * a.inv_hidden + a.eps);
  most = row_amax(most, part[1], 32, 0) * inv;
  pdl_trigger();
  const float scale = amax_nan(1e-12f, most, 0.f) / 127.f, by = 1.f / scale;
  if (threadIdx.x == 0) a.scales[row] = scale;
  for (int v = threadIdx.x; v < a.nvec; v += 1024) {
    const int64_t at = static_cast<int64_t>(v) * Vec<VEC>::kElems;
    load(at);
    if (a.r) st_global<VEC>(a.t + row * a.t_stride + at, rounded);
#pragma unroll
    for (int e = 0; e < P; ++e) y[e] = __fmul2_rn(y[e], make_float2(inv, inv));
    store_codes<VEC>(a.q + row * a.q_stride + at, y, by);
  }
}

// ---------------------------------------------------------------------------
// The product.

// Rows of bytes copied to rows on 32-byte boundaries, zeros behind them.
struct ByteCopy {
  uint8_t* dst;
  const uint8_t* src;
  int64_t dst_ld, src_ld, rows, cols;
};
struct ByteCopies {
  ByteCopy c[2];
};

// A warp copies kByteSpan bytes of a row at a time: the words of memory that they
// lie in, all of a lane's loads in flight, put together with the next lane's.  Half
// of a grid that stays resident takes each operand.  (64 x 3287 and 15814 x 3287,
// nothing in L2: 30 us; 96 with a span of 512 bytes a warp and its end.)
constexpr int kByteSpan = 1024;

__device__ __forceinline__ void copy_byte_span(const ByteCopy& c, int64_t i, int64_t j0) {
  constexpr int kWords = kByteSpan / 128;
  const int lane = threadIdx.x % 32;
  const uint8_t* row = c.src + i * c.src_ld;
  const uint8_t* end = c.src + (c.rows - 1) * c.src_ld + c.cols;  // of the tensor
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 3);
  const uint8_t* from = row - shift + j0;
  uint32_t w[kWords + 1];  // words lane, 32 + lane, ...; the last one the first lane's alone
  if (from >= c.src && from + kByteSpan + 4 <= end) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(from) + lane;
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = p[32 * k];
    w[kWords] = lane == 0 ? p[32 * kWords] : 0;
  } else {
    // Words that reach out of the tensor byte by byte.
#pragma unroll 1
    for (int k = 0; k <= kWords; ++k) {
      const uint8_t* p = from + 4 * (32 * k + lane);
      uint32_t v = 0;
      if (!(k == kWords && lane > 0) && p < end && p + 4 > c.src) {
        if (p >= c.src && p + 4 <= end) {
          v = *reinterpret_cast<const uint32_t*>(p);
        } else {
          for (int b = 0; b < 4; ++b)
            if (p + b >= c.src && p + b < end) v |= static_cast<uint32_t>(p[b]) << (8 * b);
        }
      }
#pragma unroll
      for (int q = 0; q <= kWords; ++q) w[q] = q == k ? v : w[q];
    }
  }
#pragma unroll
  for (int k = 0; k < kWords; ++k) {
    // The next lane's word; behind the last lane's comes the first one's next.
    const uint32_t next = __shfl_sync(~0u, lane == 0 ? w[k + 1] : w[k], (lane + 1) % 32);
    uint32_t v = __funnelshift_r(w[k], next, 8 * shift);
    const int64_t j = j0 + 4 * (32 * k + lane), left = c.cols - j;
    if (left < 4) v = left <= 0 ? 0 : v & (0xffffffffu >> (8 * (4 - left)));
    if (j < c.dst_ld) *reinterpret_cast<uint32_t*>(c.dst + i * c.dst_ld + j) = v;
  }
}

__global__ void __launch_bounds__(256) copy_byte_rows(ByteCopies both, uint32_t x_ctas) {
  pdl_wait();
  const bool second = blockIdx.x >= x_ctas;
  const ByteCopy c = second ? both.c[1] : both.c[0];
  const uint32_t spans = static_cast<uint32_t>((c.dst_ld + kByteSpan - 1) / kByteSpan);
  if (spans > 0) {
    // Spans in the rows' order, a warp every `step`-th; row and span by steps, without
    // a division each.
    const uint32_t first = (blockIdx.x - (second ? x_ctas : 0)) * 8 + threadIdx.x / 32;
    const uint32_t step = (second ? gridDim.x - x_ctas : x_ctas) * 8;
    const uint32_t step_rows = step / spans, step_spans = step % spans;
    uint32_t span = first % spans;
    for (int64_t i = first / spans; i < c.rows;) {
      copy_byte_span(c, i, static_cast<int64_t>(span) * kByteSpan);
      i += step_rows, span += step_spans;
      if (span >= spans) span -= spans, ++i;
    }
  }
  pdl_trigger();
}

// An operand as TMA reads it: rows on 16-byte boundaries and of an even length
// (the tensor map counts pairs), or a copy of it.
class ByteRows {
 public:
  ByteRows(Workspace& ws, const void* p, int64_t rows, int64_t cols, int64_t ld)
      : src_(static_cast<const uint8_t*>(p)), rows_(rows), cols_(cols), src_ld_(ld), ld_(ld) {
    if (rows <= 1) ld_ = round_up(cols > 0 ? cols : 1, 16);
    if (rows <= 0 || cols <= 0 || (aligned(p, 16) && (rows <= 1 || ld % 16 == 0) && cols % 2 == 0)) return;
    ld_ = round_up(cols, 32);
    copies_ = true;
    copy_ = ws.take<uint8_t>(rows * ld_);
  }
  // Pairs of bytes, as the products count.
  const uint16_t* data() const { return reinterpret_cast<const uint16_t*>(copies_ ? copy_ : src_); }
  int64_t ld() const { return ld_ / 2; }
  ByteCopy copy() const { return copies_ ? ByteCopy{copy_, src_, ld_, src_ld_, rows_, cols_} : ByteCopy{}; }

 private:
  const uint8_t* src_;
  int64_t rows_, cols_, src_ld_, ld_;
  bool copies_ = false;
  uint8_t* copy_ = nullptr;
};

// Few rows (few_rows.cuh), a CTA for 16 channels.
struct FewArgs {
  FewOperands in;
  uint16_t* out;
  const float* row_scale;
  const float* channel_scale;
  const uint16_t* bias;  // or null
  int64_t out_ld;
};

template <typename T, int kTiles, int kAlign>
__global__ void __launch_bounds__(32 * kFewWarps, kTiles == 1 ? 4 : kTiles == 2 ? 3 : 2) few_int8(FewArgs a) {
  __shared__ FewSums<int8_t, kTiles, 1> sums;
  const int channel = blockIdx.x * 16;
  few_products<int8_t, kTiles, 1, kAlign>(a.in, channel, sums);
  for (int e = threadIdx.x; e < 16 * 8 * kTiles; e += 32 * kFewWarps) {
    const int c = e % 16, i = e / 16, j = channel + c;
    if (i >= a.in.rows || j >= a.in.channels) continue;
    int sum = 0;
#pragma unroll
    for (int k = 0; k < kFewWarps; ++k) sum += sums[k][i][c];
    float y = static_cast<float>(sum) * a.row_scale[i] * a.channel_scale[j];
    if (a.bias) y += unpack1<T>(a.bias[j]);
    a.out[i * a.out_ld + j] = pack1<T>(y);
  }
}

template <typename T>
struct ScaledEpilogue {
  static constexpr bool kPaired = false;
  static constexpr int kSegment = 0;
  static constexpr bool kInteger = true;
  Out16 out;
  const float* row_scale = nullptr;
  const float* channel_scale = nullptr;
  const uint16_t* bias = nullptr;  // or null

  struct Row {
    float scale;
  };
  __device__ __forceinline__ Row begin(const Lane& l, int64_t i) const { return Row{l.inside ? row_scale[i] : 0.f}; }
  // A lane reads one column's scale and hands it round: a load a chunk, its latency
  // under the tensor memory's.
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t i, int64_t j, float (&v)[kChunk]) const {
    const bool mine = j + l.lane < out.n;
    const float scale = mine ? channel_scale[j + l.lane] : 0.f;
    const float add = mine && bias ? unpack1<T>(bias[j + l.lane]) : 0.f;
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      v[k] = static_cast<float>(__float_as_int(v[k])) * r.scale * __shfl_sync(~0u, scale, k);
      if (bias) v[k] += __shfl_sync(~0u, add, k);
    }
    out.template store<T>(l, i, j, v);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
  __device__ __forceinline__ void point(int64_t i, int64_t j, float v) const {
    float y = static_cast<float>(__float_as_int(v)) * row_scale[i] * channel_scale[j];
    if (bias) y += unpack1<T>(bias[j]);
    out.p[i * out.ld + j] = pack1<T>(y);
  }
};

namespace {

// Products that few_int8 takes: rows of both operands in vectors of 16 or 8 bytes,
// and up to 8 rows; more where the weight is small, since every CTA reads all of x
// (us, few_int8 against the tiles: 28672 x 4096, 1 row 20.1 / 25.2, 8 rows 21.8 /
// 25.6, 16 rows 29 / 25.8; 6144 x 4096, 1 row 6.2 / 10.9, 16 rows 7.8 / 10.9, 24
// rows 11.8 / 10.8; 1024 x 1024, 1 row 2.2 / 4.7, 32 rows 2.8 / 4.7).
// Returns what the rows are multiples of (rows of 8 bytes would have to be copied for
// the tiles), or 0.
int few_product(const void* x, const void* w, int64_t rows, int64_t hidden, int64_t channels, int64_t x_ld, int64_t w_ld) {
  const int64_t most = rows <= 8 ? INT64_MAX : rows <= 16 ? int64_t{32} << 20 : rows <= 32 ? int64_t{8} << 20 : 0;
  if (rows < 1 || hidden < 1 || channels * hidden > most) return 0;
  for (int align : {16, 8})
    if (hidden % align == 0 && aligned(x, align) && aligned(w, align) && (rows <= 1 || x_ld % align == 0) &&
        (channels <= 1 || w_ld % align == 0))
      return align;
  return 0;
}

template <typename T, bool kNorm>
void (*quant_kernel(int vec, int vpt, int64_t threads))(QuantArgs) {
  // Two CTAs an SM, as in gated_norm.cu (4096 x 12288 with a residual: 65.6 us with one, 52.0 with two).
  if (vec == 32 && vpt == 1 && threads > 640 && threads <= 768) return quant_rows<T, 32, 1, false, kNorm, 768>;
  if (vec == 32) return vpt == 1 ? quant_rows<T, 32, 1, false, kNorm> : nullptr;
  if (vec == 16) return vpt == 1 ? quant_rows<T, 16, 1, false, kNorm> : quant_rows<T, 16, 2, false, kNorm>;
  return vpt == 1 ? quant_rows<T, 16, 1, true, kNorm> : quant_rows<T, 16, 2, true, kNorm>;
}

template <typename T>
int launch_quant(QuantArgs& a, int vec, const DeviceInfo* dev, cudaStream_t stream, unsigned flags) {
  const char* what = "rms_norm_int8";
  const int64_t elems = vec > 0 ? vec / 2 : 8;
  a.nvec = static_cast<int32_t>((a.hidden + elems - 1) / elems);
  for (int vpt = 1; vpt <= 2; ++vpt) {
    const int64_t threads = round_up((a.nvec + vpt - 1) / vpt, 32);
    const auto fn = a.w ? quant_kernel<T, true>(vec, vpt, threads) : quant_kernel<T, false>(vec, vpt, threads);
    if (!fn || threads > 1024) continue;
    a.row_threads = static_cast<int32_t>(threads);
    const int groups = threads <= 64 ? static_cast<int>(128 / threads) : 1;
    const int64_t wave = first_wave_ctas(dev, reinterpret_cast<const void*>(fn), static_cast<int>(threads) * groups) * groups;
    // Rows that start anywhere are bound by issue: more than a wave of them by two vectors
    // a thread, half the sums over threads for each (us, one / two): 3084 x 1001 10.5 / 9.5,
    // x 5001 66 / 38, 592 x 3001 7.3 / 5.9; of less than a wave 592 x 1001 3.4 / 4.3.
    if (vec == 0 && vpt == 1 && wave > 0 && a.rows > wave && 2 * round_up((a.nvec + 1) / 2, 32) <= threads) continue;
    a.wave_rows = wave > 0 && a.rows > wave ? static_cast<int32_t>(wave) : 0;
    return launch_rows(fn, dim3(static_cast<unsigned>((a.rows + groups - 1) / groups)),
                       dim3(static_cast<unsigned>(threads * groups)), stream, flags, what, a);
  }
  if (vec >= 16) {
    a.nvec = a.hidden / 8;
    return launch_rows(quant_long_rows<T, 16>, dim3(a.rows), dim3(1024), stream, flags, what, a);
  }
  a.nvec = a.hidden;
  return launch_rows(quant_long_rows<T, 2>, dim3(a.rows), dim3(1024), stream, flags, what, a);
}

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_rms_norm_int8(int8_t* out, float* scales, void* residual_out, const void* input, const void* weight,
                       const void* residual, int64_t rows, int64_t hidden, int64_t out_row_stride,
                       int64_t residual_out_row_stride, int64_t input_row_stride, int64_t residual_row_stride,
                       double eps, int dtype, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL)) return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (rows < 0 || hidden < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || hidden > kMaxExtent)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows and hidden must be at most 2^30");
  if ((residual != nullptr) != (residual_out != nullptr))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "residual and residual_out go together");
  if (rows > 1 && (out_row_stride < hidden || input_row_stride < hidden ||
                   (residual && (residual_row_stride < hidden || residual_out_row_stride < hidden))))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  if (rows > 0 && hidden == 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "hidden must be at least 1: a row of nothing has no scale");
  if (rows == 0) return ok();
  if (!out || !scales || !input) return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  for (const void* p : {static_cast<const void*>(residual_out), input, weight, residual})
    if (!aligned(p, 2)) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  if (!aligned(scales, 4)) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  if (rows == 1) out_row_stride = residual_out_row_stride = input_row_stride = residual_row_stride = hidden;
  const Extent r = extent16(residual, rows, hidden, residual_row_stride),
               t = extent16(residual_out, rows, hidden, residual_out_row_stride);
  const Extent outs[] = {extent_of(out, rows, hidden, out_row_stride, 1), extent32(scales, 1, rows, rows), t};
  const Extent ins[] = {extent16(input, rows, hidden, input_row_stride), extent16(weight, 1, hidden, hidden)};
  const bool same_r = residual_out == residual && residual_out_row_stride == residual_row_stride;
  if (!disjoint(outs, ins) || extents_overlap(outs[0], r) || extents_overlap(outs[1], r) ||
      (!same_r && extents_overlap(t, r)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors, but for residual_out == residual");
  const DeviceInfo* dev = nullptr;
  const int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  QuantArgs a{};
  a.q = out, a.scales = scales, a.t = static_cast<uint16_t*>(residual_out);
  a.x = static_cast<const uint16_t*>(input), a.r = static_cast<const uint16_t*>(residual);
  a.w = static_cast<const uint16_t*>(weight);
  a.q_stride = out_row_stride, a.t_stride = residual_out_row_stride, a.x_stride = input_row_stride;
  a.r_stride = residual_row_stride;
  a.rows = static_cast<int32_t>(rows), a.hidden = static_cast<int32_t>(hidden);
  a.eps = static_cast<float>(eps), a.inv_hidden = 1.f / static_cast<float>(hidden);
  int vec = 0;  // rows that start anywhere
  for (int v : {32, 16}) {
    auto fits = [&](const void* p, int64_t stride, int bytes) {
      return aligned(p, v * bytes / 2) && (rows <= 1 || !p || stride * bytes % (v * bytes / 2) == 0);
    };
    if (hidden * 2 % v == 0 && fits(out, out_row_stride, 1) && fits(residual_out, residual_out_row_stride, 2) &&
        fits(input, input_row_stride, 2) && fits(residual, residual_row_stride, 2) && aligned(weight, v)) {
      vec = v;
      break;
    }
  }
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == HPRN_DTYPE_BF16 ? launch_quant<__nv_bfloat16>(a, vec, dev, cs, flags)
                                  : launch_quant<__half>(a, vec, dev, cs, flags);
}

int hprn_linear_int8(void* out, const int8_t* input, const float* input_scale, const int8_t* weight,
                     const float* weight_scale, const void* bias, int64_t rows, int64_t hidden, int64_t channels,
                     int64_t out_row_stride, int64_t input_row_stride, int64_t weight_row_stride, int dtype,
                     void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (rows < 0 || hidden < 0 || channels < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || channels > kMaxExtent)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows and channels must be at most 2^30");
  if (hidden > 131071)  // (-128)^2 * 131072 = 2^31
    return fail(HPRN_ERR_INVALID_ARGUMENT, "hidden must be at most 131071: the sums are 32-bit integers");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  if ((rows > 1 && (input_row_stride < hidden || out_row_stride < channels)) ||
      (channels > 1 && weight_row_stride < hidden))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  const int few = few_product(input, weight, rows, hidden, channels, input_row_stride, weight_row_stride);
  Workspace ws(workspace, *workspace_bytes);
  const ByteRows x(ws, input, few ? 0 : rows, hidden, input_row_stride);
  const ByteRows w(ws, weight, few ? 0 : channels, hidden, weight_row_stride);
  const int64_t pairs = (hidden + 1) / 2;
  const PlannedProduct<false, true, true> product(ws, rows, channels, pairs);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (rows == 0 || channels == 0) return ok();
  if (!out || !input_scale || !weight_scale || (hidden > 0 && (!input || !weight)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(out, 2) || !aligned(input_scale, 4) || !aligned(weight_scale, 4) || !aligned(bias, 2))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(out, rows, channels, out_row_stride)};
  const Extent ins[] = {extent_of(input, rows, hidden, input_row_stride, 1),
                        extent_of(weight, channels, hidden, weight_row_stride, 1),
                        extent32(input_scale, 1, rows, rows), extent32(weight_scale, 1, channels, channels),
                        extent16(bias, 1, channels, channels)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const char* what = "linear_int8";
  const ByteCopies copies{{x.copy(), w.copy()}};
  auto ctas_of = [&](const ByteCopy& c) {
    const int64_t n = (c.rows * ((c.dst_ld + kByteSpan - 1) / kByteSpan) + 7) / 8, most = 6 * dev->sm_count;
    return static_cast<uint32_t>(n < most ? n : most);
  };
  const uint32_t x_ctas = ctas_of(copies.c[0]), w_ctas = ctas_of(copies.c[1]);
  if (x_ctas + w_ctas > 0) {
    st = launch_rows(copy_byte_rows, dim3(x_ctas + w_ctas), dim3(256), cs, flags, what, copies, x_ctas);
    if (st != HPRN_OK) return st;
  }
  auto launch = [&](auto t) {
    using T = decltype(t);
    if (few) {
      FewArgs f{};
      f.in.x = reinterpret_cast<const uint8_t*>(input), f.in.w = reinterpret_cast<const uint8_t*>(weight);
      f.in.x_ld = rows > 1 ? input_row_stride : hidden, f.in.w_ld = channels > 1 ? weight_row_stride : hidden;
      f.in.rows = static_cast<int32_t>(rows), f.in.bytes = static_cast<int32_t>(hidden);
      f.in.channels = static_cast<int32_t>(channels);
      f.out = static_cast<uint16_t*>(out), f.out_ld = out_row_stride;
      f.row_scale = input_scale, f.channel_scale = weight_scale, f.bias = static_cast<const uint16_t*>(bias);
      const auto kernel = [&](auto align) {
        constexpr int kAlign = decltype(align)::value;
        return rows <= 8 ? few_int8<T, 1, kAlign> : rows <= 16 ? few_int8<T, 2, kAlign> : few_int8<T, 4, kAlign>;
      };
      const auto fn = few == 16 ? kernel(std::integral_constant<int, 16>{}) : kernel(std::integral_constant<int, 8>{});
      f.in.first_wave = static_cast<int32_t>(first_wave_ctas(dev, reinterpret_cast<const void*>(fn), 32 * kFewWarps));
      return launch_rows(fn, dim3(static_cast<unsigned>((channels + 15) / 16)), dim3(32 * kFewWarps), cs, flags, what, f);
    }
    Product q;
    q.a = {x.data(), x.ld()};
    q.b = {w.data(), w.ld()};
    q.m = rows, q.n = channels, q.depth = pairs;
    ScaledEpilogue<T> e;
    e.out = Out16(out, out_row_stride, channels);
    e.row_scale = input_scale, e.channel_scale = weight_scale, e.bias = static_cast<const uint16_t*>(bias);
    return product.template launch<int8_t>(q, e, cs, flags, what);
  };
  return dtype == HPRN_DTYPE_BF16 ? launch(__nv_bfloat16{}) : launch(__half{});
}

}  // extern "C"
