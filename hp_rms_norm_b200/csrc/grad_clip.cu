// The global 2-norm of many gradient tensors, and their clipping:
//   norm = sqrt(sum over every element of every tensor of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// The tensors' addresses, sizes and types travel as a kernel parameter (no
// copy to the device, so the calls can be captured in a CUDA graph), up to
// kMaxTensors a launch.  Every tensor is cut into chunks; a chunk's CTA finds
// its tensor by bisection over the first-chunk numbers.  A chunk's squares are
// summed in fp32 (eight sums a thread, at most 32 terms each), the chunks' sums
// in fp64, in an order that depends on the sizes and alignments alone, so the
// norm repeats bit for bit.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

// Tables of two sizes: a launch copies its parameters, which for the large one
// costs the host some 3 us.
constexpr int kMaxTensors = 400, kFewTensors = 50;
constexpr int kClipThreads = 256;
// Elements of a chunk: as many as give every SM some 8 chunks, within bounds
// that keep a chunk's work above its start (looking up its tensor; 4096
// elements took 5.8 us where 16384 take 4.1 on 3.5 million) and a large model's
// chunks short enough to end together.
constexpr int64_t kLeastChunk = 16384, kMostChunk = 65536;
inline int64_t chunk_elems(int64_t total) {
  const int64_t c = round_up(total / (148 * 8) + 1, 2048);
  return c < kLeastChunk ? kLeastChunk : c > kMostChunk ? kMostChunk : c;
}

struct GradEntry {
  const void* in;
  void* out;
  int64_t cols;  // elements per row; rows * cols in all
  int64_t in_stride, out_stride;
  int64_t count;
  int64_t first_chunk;
  int32_t in_type, out_type;
};

template <int N>
struct GradTable {
  static constexpr int kSize = N;
  int64_t chunk;  // elements
  int32_t n;
  GradEntry t[N];
};

template <int N>
__device__ __forceinline__ const GradEntry& find_entry(const GradTable<N>& g, int64_t chunk) {
  int lo = 0, hi = g.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (g.t[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return g.t[lo];
}

// Element types by hprn_dtype.
template <int TYPE>
struct Elem;
template <>
struct Elem<HPRN_DTYPE_BF16> {
  using Raw = uint16_t;
  static constexpr int kVec = 8;  // elements of a 16-byte vector
  static __device__ __forceinline__ float get(Raw r) { return unpack1<__nv_bfloat16>(r); }
  static __device__ __forceinline__ Raw put(float f) { return pack1<__nv_bfloat16>(f); }
};
template <>
struct Elem<HPRN_DTYPE_FP16> {
  using Raw = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(Raw r) { return unpack1<__half>(r); }
  static __device__ __forceinline__ Raw put(float f) { return pack1<__half>(f); }
};
template <>
struct Elem<HPRN_DTYPE_FP32> {
  using Raw = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(Raw r) { return r; }
  static __device__ __forceinline__ Raw put(float f) { return f; }
};

// Calls f(integral_constant<type>) for the type code.
template <typename F>
__device__ __forceinline__ void with_type(int type, F&& f) {
  if (type == HPRN_DTYPE_BF16) f(std::integral_constant<int, HPRN_DTYPE_BF16>{});
  else if (type == HPRN_DTYPE_FP16) f(std::integral_constant<int, HPRN_DTYPE_FP16>{});
  else f(std::integral_constant<int, HPRN_DTYPE_FP32>{});
}

// Eight elements as two or one 16-byte vectors.
template <int TYPE>
__device__ __forceinline__ void load8(const typename Elem<TYPE>::Raw* p, float (&v)[8]) {
  if constexpr (TYPE == HPRN_DTYPE_FP32) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    using T = typename std::conditional<TYPE == HPRN_DTYPE_BF16, __nv_bfloat16, __half>::type;
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = unpack2<T>(w[k]);
      v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
  }
}

template <int TYPE>
__device__ __forceinline__ void store8(typename Elem<TYPE>::Raw* p, const float (&v)[8]) {
  if constexpr (TYPE == HPRN_DTYPE_FP32) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]));
  } else {
    using T = typename std::conditional<TYPE == HPRN_DTYPE_BF16, __nv_bfloat16, __half>::type;
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                   pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])));
  }
}

// Elements before p's next 16-byte boundary.
template <int TYPE>
__device__ __forceinline__ int64_t ahead(const typename Elem<TYPE>::Raw* p) {
  return static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(*p);
}

// Where element k of a tensor lies.
__device__ __forceinline__ int64_t place(int64_t k, int64_t cols, int64_t stride) {
  return stride == cols ? k : k / cols * stride + k % cols;
}

// A chunk of a tensor whose rows have gaps: eight sums as below, row and column
// stepping along instead of a division an element.  A function of its own:
// inlined, it cost the dense loop a fifth (77 million bf16: 39.7 us, 31.7).
template <int TYPE>
__device__ __noinline__ float strided_squares(const GradEntry& e, int64_t lo, int64_t hi) {
  const typename Elem<TYPE>::Raw* p = static_cast<const typename Elem<TYPE>::Raw*>(e.in);
  float s[8] = {};
  const int64_t row_step = kClipThreads / e.cols, col_step = kClipThreads % e.cols;
  int64_t k = lo + threadIdx.x, row = k / e.cols, col = k % e.cols;
  while (k < hi) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (k >= hi) break;
      const float v = Elem<TYPE>::get(p[row * e.in_stride + col]);
      s[u] = fmaf(v, v, s[u]);
      k += kClipThreads, row += row_step, col += col_step;
      if (col >= e.cols) col -= e.cols, ++row;
    }
  }
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// A contiguous chunk is read in groups of eight elements from the first
// 16-byte boundary on, four groups in flight a thread; its ends one by one.
constexpr int kInFlight = 4;

template <int TYPE>
__device__ __forceinline__ float chunk_squares(const GradEntry& e, int64_t lo, int64_t hi) {
  using Raw = typename Elem<TYPE>::Raw;
  const Raw* p = static_cast<const Raw*>(e.in);
  float s[8] = {};
  auto one = [&](int64_t k) {
    const float v = Elem<TYPE>::get(p[place(k, e.cols, e.in_stride)]);
    s[0] = fmaf(v, v, s[0]);
  };
  if (e.in_stride != e.cols) return strided_squares<TYPE>(e, lo, hi);
  const int64_t first = min(lo + ahead<TYPE>(p + lo), hi), groups = (hi - first) / 8;
  for (int64_t g = threadIdx.x; g < groups; g += kClipThreads * kInFlight) {
    float v[kInFlight][8];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (g + u * kClipThreads < groups) load8<TYPE>(p + first + (g + u * kClipThreads) * 8, v[u]);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (g + u * kClipThreads < groups) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = fmaf(v[u][k], v[u][k], s[k]);
      }
  }
  for (int64_t k = lo + threadIdx.x; k < first; k += kClipThreads) one(k);
  for (int64_t k = first + groups * 8 + threadIdx.x; k < hi; k += kClipThreads) one(k);
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

template <int N>
__global__ void __launch_bounds__(kClipThreads) grad_square_sums(const __grid_constant__ GradTable<N> g,
                                                                 float* partial) {
  __shared__ float part[kClipThreads / 32];
  const GradEntry& e = find_entry(g, blockIdx.x);
  const int64_t lo = (blockIdx.x - e.first_chunk) * g.chunk;
  const int64_t hi = min(lo + g.chunk, e.count);
  pdl_wait();
  float s = 0.f;
  with_type(e.in_type, [&](auto t) { s = chunk_squares<decltype(t)::value>(e, lo, hi); });
  pdl_trigger();
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kClipThreads / 32; ++k) s += part[k];
    partial[blockIdx.x] = s;
  }
}

// The root of the sum of n partial sums, by THREADS threads, in the order of
// 1024 of them: the same bits whichever kernel joins them.  Thread 0 has it.
template <int THREADS>
__device__ __forceinline__ float join_norm(const float* partial, int64_t n) {
  constexpr int kShares = 1024 / THREADS;
  __shared__ double part[32];
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int v = 0; v < kShares; ++v) {
    const int share = threadIdx.x + v * THREADS;
    double s = 0.0;
#pragma unroll 8
    for (int64_t k = share; k < n; k += 1024) s += static_cast<double>(partial[k]);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) part[share / 32] = s;
  }
  __syncthreads();
  double s = part[lane];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return static_cast<float>(sqrt(s));
}

__global__ void __launch_bounds__(1024) grad_norm_join(const float* partial, int64_t n, float* norm) {
  pdl_wait();
  pdl_trigger();
  const float r = join_norm<1024>(partial, n);
  if (threadIdx.x == 0) *norm = r;
}

template <int IN, int OUT>
__device__ __forceinline__ void chunk_scale(const GradEntry& e, int64_t lo, int64_t hi, float f) {
  using RawIn = typename Elem<IN>::Raw;
  using RawOut = typename Elem<OUT>::Raw;
  const RawIn* p = static_cast<const RawIn*>(e.in);
  RawOut* q = static_cast<RawOut*>(e.out);
  auto one = [&](int64_t k) {
    q[place(k, e.cols, e.out_stride)] = Elem<OUT>::put(Elem<IN>::get(p[place(k, e.cols, e.in_stride)]) * f);
  };
  const int64_t first = min(lo + ahead<IN>(p + lo), hi);
  if (e.in_stride != e.cols || e.out_stride != e.cols || (reinterpret_cast<uintptr_t>(q + first) & 15) != 0) {
    for (int64_t k = lo + threadIdx.x; k < hi; k += kClipThreads) one(k);
    return;
  }
  const int64_t groups = (hi - first) / 8;
  for (int64_t g = threadIdx.x; g < groups; g += kClipThreads * kInFlight) {
    float v[kInFlight][8];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (g + u * kClipThreads < groups) load8<IN>(p + first + (g + u * kClipThreads) * 8, v[u]);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (g + u * kClipThreads < groups) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[u][k] *= f;
        store8<OUT>(q + first + (g + u * kClipThreads) * 8, v[u]);
      }
  }
  for (int64_t k = lo + threadIdx.x; k < first; k += kClipThreads) one(k);
  for (int64_t k = first + groups * 8 + threadIdx.x; k < hi; k += kClipThreads) one(k);
}

// The chunks are taken last to first: the norm's pass read the last ones last,
// so they are the ones L2 still holds.
//
// With `partial`, every CTA joins the norm's `parts` partial sums for itself and
// one writes it down: a launch less where there are few (33 tensors of 3.5
// million gradients 18.9 us a call instead of 20.5).
constexpr int64_t kFewParts = 2048;

template <int N>
__global__ void __launch_bounds__(kClipThreads)
    grad_scale(const __grid_constant__ GradTable<N> g, const float* partial, int64_t parts, float* norm,
               float max_norm) {
  const int64_t chunk = static_cast<int64_t>(gridDim.x) - 1 - blockIdx.x;
  const GradEntry& e = find_entry(g, chunk);
  const int64_t lo = (chunk - e.first_chunk) * g.chunk;
  const int64_t hi = min(lo + g.chunk, e.count);
  pdl_wait();
  // min(1, .) written so that a NaN norm gives a NaN factor.
  const float length = partial ? join_norm<kClipThreads>(partial, parts) : *norm;
  if (partial && blockIdx.x == 0 && threadIdx.x == 0) *norm = length;
  const float r = max_norm / (length + 1e-6f);
  const float f = r >= 1.f ? 1.f : r;
  if (f == 1.f && e.in == e.out) return;  // in place, and nothing to change
  with_type(e.in_type, [&](auto in) {
    with_type(e.out_type, [&](auto out) { chunk_scale<decltype(in)::value, decltype(out)::value>(e, lo, hi, f); });
  });
}

namespace {

bool known_type(int t) { return t == HPRN_DTYPE_BF16 || t == HPRN_DTYPE_FP16 || t == HPRN_DTYPE_FP32; }
int64_t elem_bytes(int t) { return t == HPRN_DTYPE_FP32 ? 4 : 2; }

int check_grads(const hprn_grad* g, int64_t count, bool with_out) {
  if (count < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "count must be >= 0");
  if (count > 0 && !g) return fail(HPRN_ERR_INVALID_ARGUMENT, "null gradient array");
  for (int64_t k = 0; k < count; ++k) {
    const hprn_grad& e = g[k];
    if (!known_type(e.dtype) || (with_out && !known_type(e.out_dtype)))
      return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16, kBFloat16 or kFloat");
    if (e.rows < 0 || e.cols < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
    if (e.rows == 0 || e.cols == 0) continue;
    if (e.rows > (int64_t{1} << 46) / e.cols)
      return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor too large");
    if (!e.grad || (with_out && !e.out)) return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned(e.grad, static_cast<int>(elem_bytes(e.dtype))) ||
        (with_out && !aligned(e.out, static_cast<int>(elem_bytes(e.out_dtype)))))
      return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
    if (e.rows > 1 && (e.row_stride < e.cols || (with_out && e.out_row_stride < e.cols)))
      return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
    if (with_out) {
      const bool same = e.out == e.grad && e.dtype == e.out_dtype &&
                        (e.rows == 1 || e.row_stride == e.out_row_stride);
      if (!same && extents_overlap(extent_of(e.grad, e.rows, e.cols, e.row_stride, elem_bytes(e.dtype)),
                           extent_of(e.out, e.rows, e.cols, e.out_row_stride, elem_bytes(e.out_dtype))))
        return fail(HPRN_ERR_INVALID_ARGUMENT,
                    "out must be the gradient itself or must not overlap it");
    }
  }
  return HPRN_OK;
}

int64_t total_of(const hprn_grad* g, int64_t count) {
  int64_t n = 0;
  for (int64_t k = 0; k < count; ++k) n += g[k].rows * g[k].cols;
  return n;
}
int64_t chunks_of(const hprn_grad& e, int64_t chunk) { return (e.rows * e.cols + chunk - 1) / chunk; }

// Calls f(table, chunks) for every launch's worth of tensors.
template <int N, typename F>
int for_tables_of(const hprn_grad* g, int64_t count, F&& f) {
  GradTable<N> table;
  table.n = 0;
  table.chunk = chunk_elems(total_of(g, count));
  int64_t chunks = 0;
  for (int64_t k = 0; k < count; ++k) {
    const int64_t c = chunks_of(g[k], table.chunk);
    if (c == 0) continue;
    if (c > 2147483647) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor too large");
    if (table.n == N || chunks + c > 2147483647) {
      const int st = f(table, chunks);
      if (st != HPRN_OK) return st;
      table.n = 0, chunks = 0;
    }
    GradEntry& e = table.t[table.n++];
    e.in = g[k].grad, e.out = g[k].out;
    e.cols = g[k].cols, e.count = g[k].rows * g[k].cols;
    e.in_stride = g[k].rows == 1 ? g[k].cols : g[k].row_stride;
    e.out_stride = g[k].rows == 1 ? g[k].cols : g[k].out_row_stride;
    e.in_type = g[k].dtype, e.out_type = g[k].out_dtype;
    e.first_chunk = chunks;
    chunks += c;
  }
  return table.n > 0 ? f(table, chunks) : HPRN_OK;
}
template <typename F>
int for_tables(const hprn_grad* g, int64_t count, F&& f) {
  return count <= kFewTensors ? for_tables_of<kFewTensors>(g, count, f) : for_tables_of<kMaxTensors>(g, count, f);
}

}  // namespace
}  // namespace hprn

namespace hprn {
namespace {

// The squares' pass; leaves one partial sum a chunk.
int launch_squares(const hprn_grad* grads, int64_t count, float* partial, cudaStream_t cs, unsigned flags,
                   const char* what) {
  int64_t at = 0;
  return for_tables(grads, count, [&](const auto& t, int64_t chunks) {
    float* part = partial + at;
    at += chunks;
    constexpr int kTensors = std::decay_t<decltype(t)>::kSize;
    return launch_rows(grad_square_sums<kTensors>, dim3(static_cast<unsigned>(chunks)), dim3(kClipThreads), cs,
                       flags, what, t, part);
  });
}

int launch_scale(const hprn_grad* grads, int64_t count, const float* partial, int64_t parts, float* norm,
                 double max_norm, cudaStream_t cs, unsigned flags, const char* what) {
  return for_tables(grads, count, [&](const auto& t, int64_t chunks) {
    constexpr int kTensors = std::decay_t<decltype(t)>::kSize;
    return launch_rows(grad_scale<kTensors>, dim3(static_cast<unsigned>(chunks)), dim3(kClipThreads), cs, flags,
                       what, t, partial, parts, norm, static_cast<float>(max_norm));
  });
}

int64_t parts_of(const hprn_grad* grads, int64_t count) {
  const int64_t chunk = chunk_elems(total_of(grads, count));
  int64_t total = 0;
  for (int64_t k = 0; k < count; ++k) total += chunks_of(grads[k], chunk);
  return total;
}

// hprn_grad_norm, and with `clip` the scaling after it.
int norm_and_clip(float* norm, const hprn_grad* grads, int64_t count, bool clip, double max_norm,
                  void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags, const char* what) {
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  if (clip && !(max_norm >= 0)) return fail(HPRN_ERR_INVALID_ARGUMENT, "max_norm must be >= 0");
  int st = check_grads(grads, count, clip);
  if (st != HPRN_OK) return st;
  const int64_t parts = parts_of(grads, count);
  Workspace ws(workspace, *workspace_bytes);
  float* partial = ws.take<float>(parts);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (!norm) return fail(HPRN_ERR_INVALID_ARGUMENT, "null norm pointer");
  if (!aligned(norm, 4)) return fail(HPRN_ERR_INVALID_ARGUMENT, "norm must be 4-byte aligned");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if ((st = launch_squares(grads, count, partial, cs, flags, what)) != HPRN_OK) return st;
  // In place, a joining CTA must not find a gradient already scaled: the
  // partial sums are complete before the first of them starts.
  if (clip && parts > 0 && parts <= kFewParts)
    return launch_scale(grads, count, partial, parts, norm, max_norm, cs, flags, what);
  st = launch_rows(grad_norm_join, dim3(1), dim3(1024), cs, flags, what, partial, parts, norm);
  if (st != HPRN_OK || !clip) return st;
  st = launch_scale(grads, count, nullptr, 0, norm, max_norm, cs, flags, what);
  return st == HPRN_OK ? ok() : st;
}

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_grad_norm(float* norm, const hprn_grad* grads, int64_t count, void* workspace,
                   int64_t* workspace_bytes, void* stream, unsigned flags) {
  return hprn::norm_and_clip(norm, grads, count, false, 0.0, workspace, workspace_bytes, stream, flags,
                             "grad_norm");
}

int hprn_clip_grad_norm(float* norm, const hprn_grad* grads, int64_t count, double max_norm, void* workspace,
                        int64_t* workspace_bytes, void* stream, unsigned flags) {
  return hprn::norm_and_clip(norm, grads, count, true, max_norm, workspace, workspace_bytes, stream, flags,
                             "clip_grad_norm");
}

int hprn_grad_clip(const hprn_grad* grads, int64_t count, const float* norm, double max_norm,
                   void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (!(max_norm >= 0)) return fail(HPRN_ERR_INVALID_ARGUMENT, "max_norm must be >= 0");
  int st = check_grads(grads, count, true);
  if (st != HPRN_OK) return st;
  if (count == 0) return ok();
  if (!norm) return fail(HPRN_ERR_INVALID_ARGUMENT, "null norm pointer");
  if (!aligned(norm, 4)) return fail(HPRN_ERR_INVALID_ARGUMENT, "norm must be 4-byte aligned");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  st = launch_scale(grads, count, nullptr, 0, const_cast<float*>(norm), max_norm,
                    static_cast<cudaStream_t>(stream), flags, "grad_clip");
  return st == HPRN_OK ? ok() : st;
}

}  // extern "C"
