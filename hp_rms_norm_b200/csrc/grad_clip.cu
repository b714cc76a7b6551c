// The global 2-norm of many gradient tensors, and their clipping:
//   norm = sqrt(sum over every element of every tensor of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// The tensors' addresses, sizes and types travel as a kernel parameter (no
// copy to the device, so the calls can be captured in a CUDA graph), up to
// kMaxTensors a launch.  Every tensor is cut into chunks of kChunkElems
// elements; a chunk's CTA finds its tensor by bisection over the first-chunk
// numbers.  A chunk's squares are summed in fp32 (at most kChunkElems / threads
// in a row per thread), the chunks' sums in fp64, in an order that depends on
// the sizes alone, so the norm repeats bit for bit.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

constexpr int kMaxTensors = 400;
constexpr int64_t kChunkElems = 16384;
constexpr int kClipThreads = 256;

struct GradEntry {
  const void* in;
  void* out;
  int64_t cols;  // elements per row; rows * cols in all
  int64_t in_stride, out_stride;
  int64_t count;
  int64_t first_chunk;
  int32_t in_type, out_type;
};

struct GradTable {
  GradEntry t[kMaxTensors];
  int32_t n;
};

__device__ __forceinline__ const GradEntry& find_entry(const GradTable& g, int64_t chunk) {
  int lo = 0, hi = g.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (g.t[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return g.t[lo];
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int type) {
  if (type == HPRN_DTYPE_FP32) return static_cast<const float*>(p)[i];
  const uint16_t h = static_cast<const uint16_t*>(p)[i];
  return type == HPRN_DTYPE_BF16 ? unpack1<__nv_bfloat16>(h) : unpack1<__half>(h);
}

__device__ __forceinline__ void store_from_f32(void* p, int64_t i, int type, float v) {
  if (type == HPRN_DTYPE_FP32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = type == HPRN_DTYPE_BF16 ? pack1<__nv_bfloat16>(v) : pack1<__half>(v);
}

__global__ void __launch_bounds__(kClipThreads) grad_square_sums(const __grid_constant__ GradTable g,
                                                                 float* partial) {
  __shared__ float part[kClipThreads / 32];
  pdl_wait();
  const GradEntry& e = find_entry(g, blockIdx.x);
  const int64_t lo = (blockIdx.x - e.first_chunk) * kChunkElems;
  const int64_t hi = min(lo + kChunkElems, e.count);
  float s = 0.f;
  for (int64_t k = lo + threadIdx.x; k < hi; k += kClipThreads) {
    const int64_t at = e.in_stride == e.cols ? k : k / e.cols * e.in_stride + k % e.cols;
    const float v = load_as_f32(e.in, at, e.in_type);
    s = fmaf(v, v, s);
  }
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kClipThreads / 32; ++k) s += part[k];
    partial[blockIdx.x] = s;
  }
}

__global__ void __launch_bounds__(1024) grad_norm_join(const float* partial, int64_t n, float* norm) {
  __shared__ double part[32];
  pdl_wait();
  double s = 0.0;
  for (int64_t k = threadIdx.x; k < n; k += 1024) s += static_cast<double>(partial[k]);
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  s = part[threadIdx.x];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(s));
}

__global__ void __launch_bounds__(kClipThreads) grad_scale(const __grid_constant__ GradTable g,
                                                           const float* norm, float max_norm) {
  pdl_wait();
  // min(1, .) written so that a NaN norm gives a NaN factor.
  const float q = max_norm / (*norm + 1e-6f);
  const float f = q >= 1.f ? 1.f : q;
  const GradEntry& e = find_entry(g, blockIdx.x);
  if (f == 1.f && e.in == e.out) return;  // in place, and nothing to change
  const int64_t lo = (blockIdx.x - e.first_chunk) * kChunkElems;
  const int64_t hi = min(lo + kChunkElems, e.count);
  for (int64_t k = lo + threadIdx.x; k < hi; k += kClipThreads) {
    const int64_t at = e.in_stride == e.cols ? k : k / e.cols * e.in_stride + k % e.cols;
    const int64_t to = e.out_stride == e.cols ? k : k / e.cols * e.out_stride + k % e.cols;
    store_from_f32(e.out, to, e.out_type, load_as_f32(e.in, at, e.in_type) * f);
  }
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

int64_t chunks_of(const hprn_grad& e) {
  return e.rows == 0 || e.cols == 0 ? 0 : (e.rows * e.cols + kChunkElems - 1) / kChunkElems;
}

// Calls f(table, chunks) for every launch's worth of tensors.
template <typename F>
int for_tables(const hprn_grad* g, int64_t count, F&& f) {
  GradTable table;
  table.n = 0;
  int64_t chunks = 0;
  for (int64_t k = 0; k < count; ++k) {
    const int64_t c = chunks_of(g[k]);
    if (c == 0) continue;
    if (c > 2147483647) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor too large");
    if (table.n == kMaxTensors || chunks + c > 2147483647) {
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

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_grad_norm(float* norm, const hprn_grad* grads, int64_t count, void* workspace,
                   int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  int st = check_grads(grads, count, false);
  if (st != HPRN_OK) return st;
  int64_t total = 0;
  for (int64_t k = 0; k < count; ++k) total += chunks_of(grads[k]);
  Workspace ws(workspace, *workspace_bytes);
  float* partial = ws.take<float>(total);
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
  int64_t at = 0;
  st = for_tables(grads, count, [&](const GradTable& t, int64_t chunks) {
    float* part = partial + at;
    at += chunks;
    return launch_rows(grad_square_sums, dim3(static_cast<unsigned>(chunks)), dim3(kClipThreads), cs, flags,
                       "grad_norm", t, part);
  });
  if (st != HPRN_OK) return st;
  return launch_rows(grad_norm_join, dim3(1), dim3(1024), cs, flags, "grad_norm", partial, total, norm);
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
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  st = for_tables(grads, count, [&](const GradTable& t, int64_t chunks) {
    return launch_rows(grad_scale, dim3(static_cast<unsigned>(chunks)), dim3(kClipThreads), cs, flags,
                       "grad_clip", t, norm, static_cast<float>(max_norm));
  });
  return st == HPRN_OK ? ok() : st;
}

}  // extern "C"
