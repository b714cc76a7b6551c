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

// Rows copied to aligned rows, their padding filled with zeros.  A warp copies
// kSpan elements of a row at a time, all of a lane's loads in flight: 16 bytes
// each where the rows start on 16-byte boundaries, else pairs of 2-byte loads,
// neighbouring lanes neighbouring pairs.
struct RowCopy {
  uint16_t* dst;
  int64_t dst_ld;
  const uint16_t* src;
  int64_t src_ld, rows, cols;
  bool vectors;
  int64_t spans;  // over all rows
};
struct RowCopies {
  RowCopy c[2];
};
constexpr int kSpan = 1024;

__global__ void __launch_bounds__(256) copy_rows(RowCopies both) {
  pdl_wait();
  const int lane = threadIdx.x % 32;
  const int64_t all = both.c[0].spans + both.c[1].spans;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; e < all;
       e += static_cast<int64_t>(gridDim.x) * 8) {
    const bool second = e >= both.c[0].spans;
    const RowCopy& c = second ? both.c[1] : both.c[0];
    const int64_t span = second ? e - both.c[0].spans : e, per_row = (c.dst_ld + kSpan - 1) / kSpan;
    const int64_t i = span / per_row, j0 = (span - i * per_row) * kSpan;
    const uint16_t* p = c.src + i * c.src_ld;
    uint16_t* q = c.dst + i * c.dst_ld;
    const int width = static_cast<int>(min(static_cast<int64_t>(kSpan), c.dst_ld - j0));  // a multiple of 16
    const int inside = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(kSpan), c.cols - j0)));
    p += j0, q += j0;
    if (c.vectors) {
      uint4 v[kSpan / 256];
#pragma unroll
      for (int k = 0; k < kSpan / 256; ++k) {
        const int j = k * 256 + lane * 8;
        v[k] = make_uint4(0, 0, 0, 0);
        if (j + 8 <= inside) v[k] = __ldcs(reinterpret_cast<const uint4*>(p + j));
      }
#pragma unroll
      for (int k = 0; k < kSpan / 256; ++k) {
        const int j = k * 256 + lane * 8;
        if (j < width) *reinterpret_cast<uint4*>(q + j) = v[k];
      }
      // The row's last elements, where they are fewer than a vector.
      const int tail = inside & ~7;
      __syncwarp();
      if (tail + lane < inside) q[tail + lane] = p[tail + lane];
      continue;
    }
    uint32_t w[kSpan / 64];
#pragma unroll
    for (int k = 0; k < kSpan / 64; ++k) {
      const int j = k * 64 + lane * 2;
      const uint32_t lo = j < inside ? p[j] : 0;
      const uint32_t hi = j + 1 < inside ? p[j + 1] : 0;
      w[k] = lo | hi << 16;
    }
#pragma unroll
    for (int k = 0; k < kSpan / 64; ++k) {
      const int j = k * 64 + lane * 2;
      if (j < width) *reinterpret_cast<uint32_t*>(q + j) = w[k];
    }
  }
}

}  // namespace

int AlignedRows::prepare(const AlignedRows& x, const AlignedRows& w, cudaStream_t stream, unsigned flags) {
  RowCopies both = {};
  int64_t spans = 0;
  both.c[0].dst_ld = both.c[1].dst_ld = 1;
  for (int k = 0; k < (&x == &w ? 1 : 2); ++k) {
    const AlignedRows* a = k == 0 ? &x : &w;
    RowCopy& c = both.c[k];
    if (!a->copies_) continue;
    c = RowCopy{a->copy_, a->ld_, a->src_, a->src_ld_, a->rows_, a->cols_,
                tma_rows(a->src_, a->rows_, a->src_ld_), a->rows_ * ((a->ld_ + kSpan - 1) / kSpan)};
    spans += c.spans;
  }
  if (spans == 0) return HPRN_OK;
  const DeviceInfo* dev = nullptr;
  const int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  const int64_t ctas = (spans + 7) / 8, most = 32 * dev->sm_count;
  return launch_rows(copy_rows, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), stream, flags,
                     "operand copy", both);
}

// Estimated clocks of a product on 148 SMs for every tiling it can take; the
// smallest wins.  The tiles run in waves of one tile per CTA (or pair), all of
// which advance together by stages of 64 terms.  A stage costs the largest of
//   its MMAs: 2 clocks a column, 400 at least,
//   its bytes from L2 at 56 a clock per SM,
//   its share of the operands' bytes from memory (each byte once, spread evenly
//   over all stages), at 3400 a clock over the whole wave and 40 per SM, so
//   that a last wave of few tiles still costs something.
// A wave adds 1500 clocks, the last tile's epilogue 20 a column (32 where two
// accumulators make a value), splitting a sum a launch (5000) and the shares'
// traffic.  Fitted to sweeps of all tilings on a B200 (bf16, clocks at
// 1.9 GHz): one row x 4096 x 2 * 14336, 256 columns 39.0 us, in two shares
// 42.0; one row x 2056 x 50001, 192 columns 39.9, 256 columns 43.8, pairs 44.1;
// 1 x 1024 x 2 * 2816, 256 columns in four shares 7.7, whole 8.8; 512 x 4096 x
// 2 * 14336, pairs 99.3, single CTAs 108.
static Tiling search_tiling(const TilingQuery& q) {
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
    for (int cols = 256; cols >= unit * group; cols -= unit) {
      // Row-major halves of B come in blocks of 64 rows.
      if (group == 2 && !q.b_k_major && cols % 128 != 0) continue;
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
        double clocks = full * (std::max(stage, slots * memory / 3400) * depth_of + 1500) + cols * (q.paired ? 32 : 20);
        if (rest > 0) clocks += std::max(stage, rest * memory / 3400) * depth_of + 1500;
        if (splits > 1) clocks += 5000 + splits * static_cast<double>(q.m) * columns * 8 / (kSms * 30);
        if (least == 0 || clocks < least) least = clocks, best = Tiling{group, cols, splits};
      }
    }
  }
  return best;
}

// The search takes 5 to 10 us, and a call asks twice for each of its products (its
// workspace's size, then the launch), so a thread keeps the last answers by the
// sizes asked about.  One row x 4096 x 6144 in int8: 26.0 us a pass with the norm
// before it without, 23.4 with.
Tiling choose_tiling(const TilingQuery& q) {
  struct Entry {
    TilingQuery q;
    Tiling t;
  };
  constexpr int kEntries = 64;
  thread_local Entry kept[kEntries] = {};
  const uint64_t mix = (static_cast<uint64_t>(q.m) * 0x9e3779b97f4a7c15u + static_cast<uint64_t>(q.n)) *
                           0xbf58476d1ce4e5b9u +
                       static_cast<uint64_t>(q.depth) * 0x94d049bb133111ebu +
                       (q.paired * 4 + q.b_k_major * 2 + q.may_split);
  Entry& e = kept[(mix >> 32) % kEntries];
  // (An entry that holds nothing has t.group 0.)
  if (e.t.group == 0 || e.q.m != q.m || e.q.n != q.n || e.q.depth != q.depth || e.q.paired != q.paired ||
      e.q.b_k_major != q.b_k_major || e.q.may_split != q.may_split)
    e = Entry{q, search_tiling(q)};
  return e.t;
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
