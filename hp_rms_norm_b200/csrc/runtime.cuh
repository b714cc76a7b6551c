// Host-side plumbing shared by the C-ABI entry points: per-thread error
// messages, a per-device attribute cache, and small launch helpers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "hp_rms_norm_b200.h"

namespace hprn {

// Records `msg` as this thread's last error and returns `status`.
int fail(int status, const std::string& msg);
// Clears this thread's last error and returns HPRN_OK.
int ok();

// Attributes of one CUDA device, read once per device and cached.
struct DeviceInfo {
  int device = -1;
  int sm_count = 0;
  int cc_major = 0;
  int cc_minor = 0;
  int max_threads_per_sm = 0;
  int regs_per_sm = 0;
  size_t smem_per_sm = 0;
  size_t smem_per_block_optin = 0;
  size_t l2_bytes = 0;
};

// Info for the calling thread's current device; returns HPRN_OK or an error
// status (with the message recorded) when the device is not an sm_100 part.
int current_device(const DeviceInfo** out);

// CTAs of kernel `fn` that one SM of `dev` holds at once at `threads`
// threads and `smem` bytes of dynamic shared memory
// (cudaOccupancyMaxActiveBlocksPerMultiprocessor), cached per (device,
// kernel, threads, smem); 0 when the query fails.
int resident_ctas_per_sm(const DeviceInfo* dev, const void* fn, int threads, size_t smem);

// How many leading CTAs of a grid of kernel `fn` (at `threads` threads, no
// dynamic shared memory) are resident at launch, i.e. the first wave:
// resident CTAs per SM x SMs.  The kernels prefetch their first rows into L2
// ahead of the programmatic-launch wait in those CTAs only (later CTAs start
// after the preceding grid is done, so a prefetch would only repeat the
// loads' own requests).  0 when the occupancy query fails: no prefetch.
inline int64_t first_wave_ctas(const DeviceInfo* dev, const void* fn, int threads) {
  return static_cast<int64_t>(resident_ctas_per_sm(dev, fn, threads, 0)) * dev->sm_count;
}

inline bool aligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes)) == 0;
}

// The largest rows / hidden / vocabulary the matrix-product entry points take.
constexpr int64_t kMaxExtent = int64_t{1} << 30;

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A caller's workspace, handed out in 256-byte aligned pieces.  Taking pieces
// only adds up sizes, so the same code answers how much a call needs.
class Workspace {
 public:
  Workspace(void* base, int64_t bytes) : base_(static_cast<char*>(base)), bytes_(bytes) {}
  template <typename T>
  T* take(int64_t count) {
    const int64_t at = round_up(used_, 256);
    used_ = at + count * static_cast<int64_t>(sizeof(T));
    return base_ ? reinterpret_cast<T*>(base_ + at) : nullptr;
  }
  int64_t needed() const { return used_; }
  bool fits() const { return used_ == 0 || (base_ && aligned(base_, 256) && used_ <= bytes_); }

 private:
  char* base_;
  int64_t bytes_;
  int64_t used_ = 0;
};

// The bytes a [rows, cols] tensor covers; null pointers cover none.
struct Extent {
  const char* lo;
  const char* hi;
  int64_t row_stride, row_bytes;
};
inline Extent extent_of(const void* p, int64_t rows, int64_t cols, int64_t row_stride, int64_t elem) {
  const char* b = static_cast<const char*>(p);
  if (!b || rows <= 0 || cols <= 0) return Extent{nullptr, nullptr, 0, 0};
  return Extent{b, b + elem * ((rows - 1) * row_stride + cols), elem * row_stride, elem * cols};
}
inline Extent extent16(const void* p, int64_t rows, int64_t cols, int64_t row_stride) {
  return extent_of(p, rows, cols, row_stride, 2);
}
inline Extent extent32(const void* p, int64_t rows, int64_t cols, int64_t row_stride) {
  return extent_of(p, rows, cols, row_stride, 4);
}
// Two tensors that share a byte.  Ranges that overlap share none where their
// rows have one stride and interleave (column slices of one buffer).
inline bool extents_overlap(const Extent& a, const Extent& b) {
  if (!(a.lo < b.hi && b.lo < a.hi)) return false;
  if (a.row_stride != b.row_stride || a.row_stride <= 0) return true;
  const int64_t m = (((b.lo - a.lo) % a.row_stride) + a.row_stride) % a.row_stride;
  return !(m >= a.row_bytes && a.row_stride - m >= b.row_bytes);
}
// No output overlaps an input or another output.
template <size_t NO, size_t NI>
bool disjoint(const Extent (&outs)[NO], const Extent (&ins)[NI]) {
  for (size_t i = 0; i < NO; ++i) {
    for (size_t j = 0; j < NI; ++j)
      if (extents_overlap(outs[i], ins[j])) return false;
    for (size_t j = 0; j < i; ++j)
      if (extents_overlap(outs[i], outs[j])) return false;
  }
  return true;
}

// Launches a kernel that begins with pdl_wait(), with programmatic stream
// serialization where `flags` ask for it.
template <typename... P, typename... A>
int launch_rows_smem(void (*fn)(P...), dim3 grid, dim3 block, int smem, cudaStream_t stream,
                     unsigned flags, const char* what, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  if (flags & HPRN_LAUNCH_PDL) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...);
  if (e != cudaSuccess)
    return fail(HPRN_ERR_CUDA, std::string(what) + " launch failed: " + cudaGetErrorString(e));
  return ok();
}

template <typename... P, typename... A>
int launch_rows(void (*fn)(P...), dim3 grid, dim3 block, cudaStream_t stream, unsigned flags,
                const char* what, A&&... args) {
  return launch_rows_smem(fn, grid, block, 0, stream, flags, what, static_cast<A&&>(args)...);
}

// The bounded waits of a launch.  A role whose wait runs out says so in two
// places: a count on the device (hprn_wait_timeouts), and a word of host memory
// that later calls look at without waiting for the GPU.
struct Waits {
  unsigned* count;
  volatile unsigned* seen;
  uint64_t limit_ns;
  bool stall;  // test hook: nothing is loaded, so that every wait for loads runs out
};
// The current device's; an error where an earlier launch's wait ran out and
// nobody has reset the count since.
int waits_of(const DeviceInfo* dev, Waits* out, const char* what);
// Clears the word in host memory.
void forget_give_ups(const DeviceInfo* dev);

#ifdef __CUDACC__
__device__ __forceinline__ void report_give_up(const Waits& w) {
  atomicAdd(w.count, 1u);
  *w.seen = 1u;
  __threadfence_system();
}
#endif

// Raises a kernel's dynamic shared memory limit, once per device.
int allow_smem(const DeviceInfo* dev, const void* fn, int bytes, const char* what);

// TMA reads rows that start on 16-byte boundaries.
inline bool tma_rows(const void* p, int64_t rows, int64_t ld) {
  return aligned(p, 16) && (rows <= 1 || ld % 8 == 0);
}

// Reports a failed launch (cudaGetLastError after the launch) as HPRN_ERR_CUDA.
int check_launch(const char* what);

}  // namespace hprn
