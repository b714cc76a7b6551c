// Host side of the matrix products: tensor maps, aligned copies of operands
// TMA cannot read, kernel attributes.
#include "matmul.cuh"

#include <algorithm>
#include <cmath>
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

// A warp copies 256 elements of a row at a time, neighbouring lanes
// neighbouring pairs, the loads 2 bytes (the rows are not aligned) and four
// pairs in flight; the row's padding is filled with zeros.
constexpr int kCopyPairs = 4;
__global__ void __launch_bounds__(256) copy_rows(uint16_t* dst, int64_t dst_ld, const uint16_t* src,
                                                 int64_t src_ld, int64_t rows, int64_t cols) {
  pdl_wait();
  constexpr int kSpan = 64 * kCopyPairs;
  const int64_t per_row = (dst_ld + kSpan - 1) / kSpan, n = rows * per_row;
  const int lane = threadIdx.x % 32;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; e < n;
       e += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t i = e / per_row, j = (e - i * per_row) * kSpan + lane * 2;
    const uint16_t* p = src + i * src_ld + j;
    uint32_t w[kCopyPairs];
#pragma unroll
    for (int k = 0; k < kCopyPairs; ++k) {
      const uint32_t lo = j + 64 * k < cols ? p[64 * k] : 0;
      const uint32_t hi = j + 64 * k + 1 < cols ? p[64 * k + 1] : 0;
      w[k] = lo | hi << 16;
    }
#pragma unroll
    for (int k = 0; k < kCopyPairs; ++k)
      if (j + 64 * k < dst_ld) *reinterpret_cast<uint32_t*>(dst + i * dst_ld + j + 64 * k) = w[k];
  }
}

}  // namespace

int AlignedRows::prepare(cudaStream_t stream, unsigned flags) const {
  if (!copies_) return HPRN_OK;
  const DeviceInfo* dev = nullptr;
  const int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  const int64_t ctas = (rows_ * ((ld_ + 255) / 256) + 7) / 8, most = 16 * dev->sm_count;
  return launch_rows(copy_rows, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), stream, flags,
                     "operand copy", copy_, ld_, src_, src_ld_, rows_, cols_);
}

// Estimated clocks of a product on 148 SMs for every tiling it can take; the
// smallest wins.  The tiles run in waves of one tile per CTA (or pair), all of
// which advance together by stages of 64 terms.  A stage costs the largest of
//   its MMAs: 2 clocks a column, 400 at least,
//   its bytes from L2 at 56 a clock per SM,
//   its share of the operands' bytes from memory (each byte once, spread evenly
//   over all stages), at 3400 a clock over the whole wave and 40 per SM, so
//   that a last wave of few tiles still costs something.
// A wave adds 1500 clocks; splitting a sum a launch (5000) and the shares'
// traffic.  Fitted to sweeps of all tilings on a B200 (bf16, clocks at
// 1.9 GHz): one row x 4096 x 2 * 14336, 256 columns 39.0 us, in two shares
// 42.0; one row x 2056 x 50001, 192 columns 39.9, 256 columns 43.8, pairs 44.1;
// 1 x 1024 x 2 * 2816, 256 columns in four shares 7.7, whole 8.8; 512 x 4096 x
// 2 * 14336, pairs 99.3, single CTAs 108.
Tiling choose_tiling(const TilingQuery& q) {
  Tiling best{2, 256, 1};
  if (q.m <= 0 || q.n <= 0 || q.depth <= 0) return best;
  constexpr int kSms = 148;
  const double depth = static_cast<double>(q.depth), blocks = std::ceil(depth / kDepthBlock);
  const double columns = static_cast<double>(q.n) * (q.paired ? 2 : 1);
  const double bytes = (static_cast<double>(q.m) + columns) * depth * 2;
  const double a_rows = q.m < 128 ? static_cast<double>(round_up(q.m, 8)) : 128.0;
  const int unit = q.paired || !q.b_k_major ? 64 : 32;
  double least = 0;
  for (int group = 2; group >= 1; --group) {
    const int slots = kSms / group;
    for (int cols = 256; cols >= (group == 2 ? 256 : unit); cols -= unit) {
      const int c_cols = q.paired ? cols / 2 : cols;
      const double tiles = static_cast<double>((q.m + 128 * group - 1) / (128 * group)) *
                           static_cast<double>((q.n + c_cols - 1) / c_cols);
      const double mma = cols * 2 < 400 ? 400 : cols * 2;
      const double load = (a_rows + cols / group) * 128 / 56;
      const double memory = bytes / (tiles * blocks);  // of one tile's stage
      const double stage = std::max({mma, load, memory / (40 * group)});
      const int most = q.may_split ? 16 : 1;
      for (int splits = 1; splits <= most && splits * 2 <= blocks; ++splits) {
        const double items = tiles * splits, full = std::floor(items / slots), rest = items - full * slots;
        const double depth_of = std::ceil(blocks / splits);
        double clocks = full * (std::max(stage, slots * memory / 3400) * depth_of + 1500) + cols * 8;
        if (rest > 0) clocks += std::max(stage, rest * memory / 3400) * depth_of + 1500;
        if (splits > 1) clocks += 5000 + splits * static_cast<double>(q.m) * columns * 8 / (kSms * 30);
        if (least == 0 || clocks < least) least = clocks, best = Tiling{group, cols, splits};
      }
    }
  }
  return best;
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

}  // namespace hprn
