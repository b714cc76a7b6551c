// Host side of the matrix products: tensor maps, aligned copies of operands
// TMA cannot read, kernel attributes.
#include "matmul.cuh"

#include <mutex>

namespace hprn {

namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// Eight elements of the copy a thread: 16-byte stores, 2-byte loads (the rows
// are not aligned), the row's padding filled with zeros.
__global__ void __launch_bounds__(256) copy_rows(uint16_t* dst, int64_t dst_ld, const uint16_t* src,
                                                 int64_t src_ld, int64_t rows, int64_t cols) {
  pdl_wait();
  const int64_t per_row = dst_ld / 8, n = rows * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n; e += step) {
    const int64_t i = e / per_row, j = (e - i * per_row) * 8;
    Vec<16> v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = j + 2 * k < cols ? src[i * src_ld + j + 2 * k] : 0;
      const uint32_t hi = j + 2 * k + 1 < cols ? src[i * src_ld + j + 2 * k + 1] : 0;
      v.w[k] = lo | hi << 16;
    }
    st_global<16>(dst + i * dst_ld + j, v);
  }
}

}  // namespace

int AlignedRows::prepare(cudaStream_t stream, unsigned flags) const {
  if (!copies_) return HPRN_OK;
  const DeviceInfo* dev = nullptr;
  const int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  const int64_t ctas = (rows_ * (ld_ / 8) + 255) / 256, most = 16 * dev->sm_count;
  return launch_rows(copy_rows, static_cast<unsigned>(ctas < most ? ctas : most), dim3(256), stream, flags,
                     "operand copy", copy_, ld_, src_, src_ld_, rows_, cols_);
}

int encode_rows(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows,
                const char* what) {
  const EncodeFn fn = encode_fn();
  if (!fn) return fail(HPRN_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  // 16-bit elements move as raw bits; rows of one tensor need no stride.
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t unit[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p), dims, strides, box,
                        unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(HPRN_ERR_CUDA, std::string(what) + ": cuTensorMapEncodeTiled failed (" +
                                   std::to_string(static_cast<int>(r)) + ")");
  return HPRN_OK;
}

int allow_smem(const DeviceInfo* dev, const void* fn, int bytes, const char* what) {
  constexpr int kMost = 512;
  static std::mutex mu;
  static const void* done_fn[kMost];
  static int done_device[kMost];
  static int done = 0;
  std::lock_guard<std::mutex> lock(mu);
  for (int k = 0; k < done; ++k)
    if (done_fn[k] == fn && done_device[k] == dev->device) return HPRN_OK;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess)
    return fail(HPRN_ERR_CUDA, std::string(what) + ": shared memory limit: " + cudaGetErrorString(e));
  if (done < kMost) done_fn[done] = fn, done_device[done] = dev->device, ++done;
  return HPRN_OK;
}

}  // namespace hprn
