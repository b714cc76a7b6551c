// Softmax cross entropy of a linear layer over a vocabulary, without keeping
// the logits L = X W^T (X [rows, hidden], W [vocab, hidden]):
//   lse_i  = log sum_j exp(L_ij),  loss_i = lse_i - L_{i, t_i}
// and 0 for rows whose target t_i is `ignore_index`.
//
// Forward: each tile of L leaves, per row, its largest value and the sum of
// exponentials relative to it (8 bytes for a tile's columns instead of 4 per
// logit), and the logit of the row's target; a second kernel joins a row's
// tiles:  lse = M + log sum_t s_t exp(m_t - M),  M = max_t m_t.
//
// Backward, c_i the gradient of loss_i:
//   S_ij = c_i (exp(L_ij - lse_i) - [j == t_i]),  dX = S W,  dW = S^T X
// one piece of the vocabulary at a time: the piece's logits are computed again
// and leave as S (16-bit, the tensor cores' operand), dW's rows of that piece
// are complete, and dX is summed over the pieces in fp32 and rounded once.
//
// S is held as c_i / c_max (exp(L_ij - lse_i) - [j == t_i]), c_max the largest
// finite |c_i|, and the sums are multiplied by c_max.  A mean gives every row the same
// c, and then the entries that matter most, -c at the targets, would all be
// rounded to 16 bits alike and the gradients come out up to 2^-9 short or long;
// -1 is exact (8192 x 4096 x 131072, one draw of the targets: 3.5e-3 off without,
// 1.7e-3, the rounding of the outputs themselves, with it).  In fp16 S is held
// times 2^14 as well: softmax values of a large vocabulary fall below its
// smallest normal, 6e-5 (now those below 3.7e-9 c_max / |c_i| do).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "matmul.cuh"
#include "runtime.cuh"
#include "vocabulary.cuh"

namespace hprn {

struct LossEpilogue {
  static constexpr bool kPaired = false;
  static constexpr int kSegment = kLogitSegment;
  static constexpr bool kUnrolled = true;
  float2* partial = nullptr;  // [rows, parts]: {max of l, sum of exp(l - max)}
  float* target_logit = nullptr;
  const int64_t* target = nullptr;
  int64_t ignore = 0;
  int64_t parts = 0;
  int64_t vocab = 0;

  struct Row {
    float m, s;
    int64_t t;
  };
  __device__ __forceinline__ Row begin(const Lane& l, int64_t i) const {
    return Row{-INFINITY, 0.f, l.inside ? target_of(target, i, ignore, vocab) : kIgnored};
  }
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t i, int64_t j, float (&v)[kChunk]) const {
    if (j + kChunk > vocab) {
      const int left = static_cast<int>(vocab - j);
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
        if (k >= left) v[k] = -INFINITY;
    }
    const int64_t at = r.t - j;
    if (at >= 0 && at < kChunk) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < kChunk; ++k) x = at == k ? v[k] : x;
      target_logit[i] = x;
    }
    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int k = 4; k < kChunk; ++k) top[k % 4] = fmaxf(top[k % 4], v[k]);
    const float m = fmaxf(r.m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    // All so far -inf (or NaN, which fmaxf skips and the sum keeps): exp(-inf - 0) = 0.
    const float ref = m == -INFINITY ? 0.f : m;
    const float2 minus = make_float2(-ref, -ref);
    float2 s[2] = {make_float2(r.s * exp_fast(r.m - ref), 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < kChunk / 2; ++k)
      s[k % 2] = __fadd2_rn(s[k % 2], exp_fast2(__fadd2_rn(make_float2(v[2 * k], v[2 * k + 1]), minus)));
    r.m = m, r.s = (s[0].x + s[0].y) + (s[1].x + s[1].y);
  }
  __device__ __forceinline__ void end(Row& r, const Lane& l, int64_t i, int64_t part) const {
    if (l.inside) partial[i * parts + part] = make_float2(r.m, r.s);
  }
};

// Joins a row's parts, one warp a row.
__global__ void __launch_bounds__(256)
    loss_join(const float2* partial, const float* target_logit, const int64_t* target, int64_t ignore,
              int64_t rows, int64_t vocab, int64_t parts, float* loss, float* lse) {
  pdl_wait();
  const int lane = threadIdx.x % 32;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
  if (i >= rows) return;
  float m = -INFINITY, s = 0.f;
  auto join = [&](float2 p) {
    const float top = fmaxf(m, p.x);
    const float ref = top == -INFINITY ? 0.f : top;
    s = s * exp_fast(m - ref) + p.y * exp_fast(p.x - ref);
    m = top;
  };
  for (int64_t k = lane; k < parts; k += 32) join(partial[i * parts + k]);
  for (int o = 16; o > 0; o >>= 1)
    join(make_float2(__shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o)));
  if (lane != 0) return;
  if (parts == 0 && vocab > 0) m = 0.f, s = static_cast<float>(vocab);  // sums of no terms: logits 0
  const float top = m == -INFINITY ? 0.f : m, log_s = logf(s);
  lse[i] = top + log_s;
  const int64_t t = target_of(target, i, ignore, vocab);
  // The two logits first: where the target is the largest one the loss is log s,
  // which a sum with a logit of 30 would round to multiples of 2^-19.
  loss[i] = t == kIgnored    ? 0.f
            : t == kInvalid ? __int_as_float(0x7fc00000)
                            : (top - (parts > 0 ? target_logit[i] : 0.f)) + log_s;
}

template <typename T>
struct LossGradEpilogue {
  static constexpr bool kPaired = false;
  static constexpr int kSegment = kLogitSegment;
  static constexpr bool kUnrolled = false;
  Out16 s;                 // the piece's columns
  const float* lse = nullptr;
  const float* grad_loss = nullptr;
  const float* most = nullptr;  // c_max
  float held = 1.f;             // what S is held times
  const int64_t* target = nullptr;
  int64_t ignore = 0;
  int64_t vocab = 0;
  int64_t first = 0;  // the piece's first column

  struct Row {
    float c, lse;
    int64_t t;  // within the piece (or outside it)
  };
  __device__ __forceinline__ Row begin(const Lane& l, int64_t i) const {
    const int64_t t = l.inside ? target_of(target, i, ignore, vocab) : kIgnored;
    if (t == kIgnored) return Row{0.f, INFINITY, kIgnored};
    // A target outside the vocabulary has no loss: NaN, like the loss itself.
    const float c = t == kInvalid ? __int_as_float(0x7fc00000) : grad_loss[i] / *most * held;
    return Row{c, lse[i], t >= first ? t - first : kInvalid};
  }
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t i, int64_t j, float (&v)[kChunk]) const {
    const int64_t at = r.t - j;
    const bool here = at >= 0 && at < kChunk;
    if (r.t == kIgnored) {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) v[k] = 0.f;
    } else {
#pragma unroll
      for (int k = 0; k < kChunk / 2; ++k) {
        const float2 l = make_float2(v[2 * k], v[2 * k + 1]);
        const float2 p = __fmul2_rn(exp_fast2(__fadd2_rn(l, make_float2(-r.lse, -r.lse))), make_float2(r.c, r.c));
        v[2 * k] = p.x, v[2 * k + 1] = p.y;
      }
      if (here) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k)
          if (at == k) v[k] -= r.c;
      }
    }
    s.template store<T>(l, i, j, v);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
};

}  // namespace hprn

extern "C" {

int hprn_linear_cross_entropy(float* loss, float* lse, const void* input, const void* weight,
                              const int64_t* target, int64_t ignore_index, int64_t rows,
                              int64_t hidden, int64_t vocab, int64_t input_row_stride,
                              int64_t weight_row_stride, int dtype, void* workspace,
                              int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  int st = check_vocabulary(rows, hidden, vocab, dtype, flags, workspace_bytes);
  if (st != HPRN_OK) return st;
  if ((rows > 1 && input_row_stride < hidden) || (vocab > 1 && weight_row_stride < hidden))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  Workspace ws(workspace, *workspace_bytes);
  const AlignedRows x(ws, input, rows, hidden, input_row_stride, vocab);
  const AlignedRows w(ws, weight, vocab, hidden, weight_row_stride, rows);
  const PlannedProduct<false, true, true> product(ws, rows, vocab, hidden, false);
  const int64_t parts = product.parts(vocab);
  float2* partial = ws.take<float2>(parts * rows);
  float* target_logit = ws.take<float>(rows);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (rows == 0) return ok();
  if (!loss || !lse || !target || (hidden > 0 && (!input || (vocab > 0 && !weight))))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(loss, 4) || !aligned(lse, 4) || !aligned(target, 8) || !aligned(input, 2) ||
      !aligned(weight, 2))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent32(loss, 1, rows, rows), extent32(lse, 1, rows, rows)};
  const Extent ins[] = {extent16(input, rows, hidden, input_row_stride),
                      extent16(weight, vocab, hidden, weight_row_stride),
                      extent_of(target, 1, rows, rows, 8)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const char* what = "linear_cross_entropy";
  if ((st = AlignedRows::prepare(x, w, cs, flags)) != HPRN_OK) return st;
  Product q;
  q.a = {x.data(), x.ld()};
  q.b = {w.data(), w.ld()};
  q.m = rows, q.n = vocab, q.depth = hidden;
  LossEpilogue e;
  e.partial = partial, e.target_logit = target_logit, e.target = target;
  e.ignore = ignore_index, e.parts = parts, e.vocab = vocab;
  if (hidden > 0) {
    st = dtype == HPRN_DTYPE_BF16 ? product.launch_whole<__nv_bfloat16>(q, e, cs, flags, what)
                                  : product.launch_whole<__half>(q, e, cs, flags, what);
    if (st != HPRN_OK) return st;
  }
  return launch_rows(loss_join, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), cs, flags, what,
                     partial, target_logit, target, ignore_index, rows, vocab, hidden > 0 ? parts : 0, loss, lse);
}

int hprn_linear_cross_entropy_backward(void* grad_input, void* grad_weight, const float* grad_loss,
                                       const void* input, const void* weight, const int64_t* target,
                                       const float* lse, int64_t ignore_index, int64_t rows,
                                       int64_t hidden, int64_t vocab, int64_t grad_input_row_stride,
                                       int64_t grad_weight_row_stride, int64_t input_row_stride,
                                       int64_t weight_row_stride, int dtype, void* workspace,
                                       int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  int st = check_vocabulary(rows, hidden, vocab, dtype, flags, workspace_bytes);
  if (st != HPRN_OK) return st;
  if ((rows > 1 && (input_row_stride < hidden || grad_input_row_stride < hidden)) ||
      (vocab > 1 && (weight_row_stride < hidden || grad_weight_row_stride < hidden)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  Workspace ws(workspace, *workspace_bytes);
  const int64_t x_ld = round_up(hidden, 16);
  uint16_t* x = ws.take<uint16_t>(rows * x_ld);  // X without the ignored rows
  const AlignedRows w(ws, weight, vocab, hidden, weight_row_stride, rows);
  const Pieces pieces = pieces_of(rows, vocab);
  uint16_t* s = ws.take<uint16_t>(rows * pieces.cols);
  const int64_t sum_ld = round_up(hidden, kChunk);
  float* sum = pieces.count > 1 ? ws.take<float>(rows * sum_ld) : nullptr;
  float* scale = ws.take<float>(2);
  const float held = dtype == HPRN_DTYPE_FP16 ? 16384.f : 1.f;
  const PlannedProduct<false, true, true> logits(ws, rows, pieces.cols, hidden, false);
  const PlannedProduct<false, true, false> to_input(ws, rows, hidden, pieces.cols);
  const PlannedProduct<false, false, false> to_weight(ws, pieces.cols, hidden, rows);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if ((rows > 0 && (!grad_input || !grad_loss || !input || !target || !lse)) ||
      (vocab > 0 && (!grad_weight || !weight)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(grad_input, 2) || !aligned(grad_weight, 2) || !aligned(grad_loss, 4) ||
      !aligned(input, 2) || !aligned(weight, 2) || !aligned(target, 8) || !aligned(lse, 4))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                       extent16(grad_weight, vocab, hidden, grad_weight_row_stride)};
  const Extent ins[] = {extent32(grad_loss, 1, rows, rows),
                      extent16(input, rows, hidden, input_row_stride),
                      extent16(weight, vocab, hidden, weight_row_stride),
                      extent_of(target, 1, rows, rows, 8), extent32(lse, 1, rows, rows)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const char* what = "linear_cross_entropy_backward";
  if ((st = w.prepare(cs, flags)) != HPRN_OK) return st;
  if (rows > 0) {
    LossPrepareArgs a{};
    a.x = static_cast<const uint16_t*>(input), a.x_ld = input_row_stride;
    a.out = x, a.out_ld = x_ld, a.rows = rows, a.hidden = hidden;
    a.spans = (x_ld + kPrepareSpan - 1) / kPrepareSpan;
    a.vectors = tma_rows(input, rows, input_row_stride);
    a.grad_loss = grad_loss, a.target = target, a.ignore = ignore_index, a.held = held, a.scale = scale;
    const int64_t ctas = (rows * a.spans + 7) / 8, most = 16 * dev->sm_count;
    st = launch_rows(loss_grad_prepare<false>, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), cs,
                     flags, what, a);
    if (st != HPRN_OK) return st;
  }
  auto all = [&](auto t) {
    using T = decltype(t);
    int r = HPRN_OK;
    // Without a vocabulary the input's gradient is an empty sum: zero.
    const int64_t count = pieces.count > 0 ? pieces.count : 1;
    for (int64_t p = 0; p < count && r == HPRN_OK; ++p) {
      const int64_t first = p * pieces.cols;
      const int64_t cols = vocab - first < pieces.cols ? vocab - first : pieces.cols;
      const uint16_t* wp = w.data() + first * w.ld();
      Product q;
      q.a = {x, x_ld};
      q.b = {wp, w.ld()};
      q.m = rows, q.n = cols, q.depth = hidden;
      LossGradEpilogue<T> g;
      g.s = Out16(s, pieces.cols, cols), g.lse = lse, g.grad_loss = grad_loss, g.most = scale, g.held = held;
      g.target = target, g.ignore = ignore_index, g.vocab = vocab, g.first = first;
      if ((r = logits.launch_whole<T>(q, g, cs, flags, what)) != HPRN_OK) break;

      q.a = {s, pieces.cols};
      q.n = hidden, q.depth = cols;
      StoreEpilogue<T> e;
      e.out = Out16(grad_input, grad_input_row_stride, hidden);
      e.sum = sum, e.sum_ld = sum_ld, e.first = p == 0, e.last = p == count - 1;
      e.scale = rows > 0 ? scale + 1 : nullptr;
      if ((r = to_input.launch<T>(q, e, cs, flags, what)) != HPRN_OK) break;

      q.b = {x, x_ld};
      q.m = cols, q.depth = rows;
      e.out = Out16(static_cast<uint16_t*>(grad_weight) + first * grad_weight_row_stride,
                    grad_weight_row_stride, hidden);
      e.sum = nullptr, e.first = e.last = true;
      r = to_weight.launch<T>(q, e, cs, flags, what);
    }
    return r;
  };
  return dtype == HPRN_DTYPE_BF16 ? all(__nv_bfloat16{}) : all(__half{});
}

int hprn_test_loss_backward_piece(int64_t rows, int64_t hidden, int64_t vocab, int64_t piece, int64_t* out) {
  using namespace hprn;
  int64_t none = 0;
  const int st = check_vocabulary(rows, hidden, vocab, HPRN_DTYPE_BF16, 0, &none);
  if (st != HPRN_OK) return st;
  const Pieces pieces = pieces_of(rows, vocab);
  if (!out || piece < 0 || piece >= pieces.count)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "no such piece of the vocabulary");
  Workspace ws(nullptr, 0);
  const PlannedProduct<false, true, false> to_input(ws, rows, hidden, pieces.cols);
  const int64_t left = vocab - piece * pieces.cols, cols = left < pieces.cols ? left : pieces.cols;
  out[0] = pieces.count, out[1] = cols;
  out[2] = (cols + kDepthBlock - 1) / kDepthBlock, out[3] = to_input.shares(cols);
  return ok();
}

}  // extern "C"
