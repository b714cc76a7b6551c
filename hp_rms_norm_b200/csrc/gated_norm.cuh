// What the gated norm's forward and backward entry points check alike.
#pragma once

#include <stdint.h>

#include "runtime.cuh"

namespace hprn {

inline int check_block_norm(int64_t rows, int64_t hidden, int64_t rows_per_gate, int64_t gate_width, bool gate,
                            int dtype) {
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

}  // namespace hprn
