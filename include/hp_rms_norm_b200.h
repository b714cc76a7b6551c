/*
 * hp_rms_norm_b200: C ABI of the B200-native (sm_100a) fused residual-add +
 * RMSNorm and ReLU kernels.
 *
 * Everything here is plain C: device pointers, element counts and strides, a
 * dtype code and a CUDA stream handle passed as void*.  No torch types cross
 * this boundary.  The torch-extension binding (torch.ops.hp_rms_norm.*) and
 * any cgo / JNI / ctypes caller bind these same symbols.
 *
 * Conventions shared by every entry point:
 *   - All tensor pointers are device pointers on the CURRENT CUDA device of
 *     the calling thread (cudaSetDevice before calling).
 *   - Work is enqueued asynchronously on `stream` (a cudaStream_t; NULL means
 *     the legacy default stream).  Nothing synchronises; nothing allocates.
 *   - Return value: HPRN_OK (0) or a negative hprn_status code; on error no
 *     kernel was launched (except HPRN_ERR_CUDA, which reports a failed
 *     launch) and hprn_last_error() returns a message for this thread.
 *   - Strides are in ELEMENTS, between consecutive rows; elements within a
 *     row are contiguous.
 */
#ifndef HP_RMS_NORM_B200_H_
#define HP_RMS_NORM_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HPRN_VERSION 10000 /* 1.0.0 */

#if defined(__GNUC__)
#define HPRN_API __attribute__((visibility("default")))
#else
#define HPRN_API
#endif

typedef enum hprn_dtype {
  HPRN_DTYPE_BF16 = 0, /* torch.bfloat16 / __nv_bfloat16 */
  HPRN_DTYPE_FP16 = 1, /* torch.float16  / __half        */
  HPRN_DTYPE_FP32 = 2  /* torch.float32 / float: gradients of hprn_grad_* only */
} hprn_dtype;

/*
 * Launch flags for the *_ex entry points.
 *   HPRN_LAUNCH_PDL: launch with programmatic stream serialization (programmatic
 *   dependent launch).  The kernel may then be scheduled while the previous
 *   kernel on the stream is still finishing; it waits (griddepcontrol.wait)
 *   for that kernel to complete before its first memory access, so results
 *   are the same as a plain launch.  Every kernel of this library also lets
 *   its own successor be scheduled early, once all of its CTAs have issued
 *   their last store.
 */
#define HPRN_LAUNCH_PDL 1u
#define HPRN_LAUNCH_DEFAULT HPRN_LAUNCH_PDL

/* Output forms of hprn_rms_norm_out. */
typedef enum hprn_out_form {
  HPRN_OUT_SAME = 0,              /* 16-bit, the input's dtype */
  HPRN_OUT_FP8_E4M3_STATIC = 1,   /* fp8 e4m3 (OCP E4M3FN), one scale for the tensor */
  HPRN_OUT_FP8_E4M3_DYNAMIC = 2,  /* fp8 e4m3, one scale per row, written to row_scales */
  HPRN_OUT_NVFP4 = 3,             /* fp4 e2m1 + e4m3 block scales: hprn_rms_norm_nvfp4 only */
  HPRN_OUT_FP8_E4M3_GROUP = 4     /* fp8 e4m3, one scale per group: hprn_rms_norm_fp8_group only */
} hprn_out_form;

/* Activations of hprn_act_and_mul. */
typedef enum hprn_act {
  HPRN_ACT_SILU = 0,      /* a / (1 + exp(-a))                                   */
  HPRN_ACT_GELU = 1,      /* a / 2 * (1 + erf(a / sqrt(2)))                      */
  HPRN_ACT_GELU_TANH = 2  /* a / 2 * (1 + tanh(sqrt(2/pi) * (a + 0.044715 a^3))) */
} hprn_act;

typedef enum hprn_status {
  HPRN_OK = 0,
  HPRN_ERR_INVALID_ARGUMENT = -1, /* bad size, stride, null pointer, overlap */
  HPRN_ERR_UNSUPPORTED_DTYPE = -2,
  HPRN_ERR_UNSUPPORTED_DEVICE = -3, /* not an sm_100 (B200-class) device */
  HPRN_ERR_CUDA = -4                /* a CUDA runtime call or launch failed */
} hprn_status;

/*
 * Fused residual add + RMSNorm, in place:
 *
 *   residual[i, :] <- round_T(f32(input[i, :]) + f32(residual[i, :]))
 *   input[i, :]    <- round_T(f32(residual[i, :]) * f32(weight[:]) * inv_i)
 *   inv_i           = rsqrt(eps + sum_j s_ij^2 / hidden),  s_ij the fp32 sum before rounding
 *
 * for rows i in [0, rows).  input and residual must not overlap.
 *
 * Replaces the reference's torch-op implementation
 *   void rms_norm(Tensor& input, const Tensor& weight, Tensor& residual, double eps)
 *     hp_rms_norm/csrc/cuda/hp_rms_norm.cu:7-50
 * and its launcher hp_rms_norm::launch_rms_norm<T>
 *     hp_rms_norm/csrc/cuda/hp_rms_norm.cuh:562-618
 * (there `rows` is the reference's `tokens` and both strides equal hidden).
 * Unlike the reference it accepts any hidden >= 1, any 2-byte-aligned pointers
 * and independent row strides; the widest vector width the pointers, strides
 * and hidden size allow is chosen per call.
 */
HPRN_API int hprn_rms_norm(void* input, const void* weight, void* residual, int64_t rows,
                           int64_t hidden, int64_t input_row_stride, int64_t residual_row_stride,
                           double eps, int dtype, void* stream);

/*
 * Elementwise ReLU, out-of-place: out[i, :] = input[i, :] <= 0 ? +0 : input[i, :]
 * (torch.relu as computed on CUDA, bit for bit: negatives, -inf and -0.0 give
 * +0; NaNs pass through with their input bits).
 * out and input may be the same pointer (in place) but must not otherwise overlap.
 *
 * Replaces the reference's
 *   void relu(Tensor& out, const Tensor& input)
 *     hp_rms_norm/csrc/cuda/activation_kernels.cu:7-39
 * and hp_rms_norm::launch_relu<T> hp_rms_norm/csrc/cuda/activation_kernels.cuh:122-145.
 * (The reference kernel copies input to out without applying max(x, 0) and
 * drops the row tail when hidden * 2 is not a multiple of 256; this entry point
 * applies ReLU to every element.)
 */
HPRN_API int hprn_relu(void* out, const void* input, int64_t rows, int64_t hidden,
                       int64_t out_row_stride, int64_t input_row_stride, int dtype, void* stream);

/*
 * hprn_rms_norm and hprn_relu with explicit launch flags (HPRN_LAUNCH_*; 0 for
 * a plain launch).  The plain entry points use HPRN_LAUNCH_DEFAULT.
 * (Extensions of the reference's fixed launch: FlashInfer-style enable_pdl.)
 */
HPRN_API int hprn_rms_norm_ex(void* input, const void* weight, void* residual, int64_t rows,
                              int64_t hidden, int64_t input_row_stride,
                              int64_t residual_row_stride, double eps, int dtype, void* stream,
                              unsigned flags);
HPRN_API int hprn_relu_ex(void* out, const void* input, int64_t rows, int64_t hidden,
                          int64_t out_row_stride, int64_t input_row_stride, int dtype,
                          void* stream, unsigned flags);

/*
 * RMSNorm with or without the residual add, into a separate output, 16-bit or
 * fp8 (an extension past the reference, whose only form is hprn_rms_norm's):
 *
 *   residual == NULL (plain RMSNorm):  s_j = f32(input[i, j])
 *   residual != NULL (fused add):      s_j = f32(input[i, j]) + f32(residual[i, j]),
 *                                      residual[i, j] <- round_T(s_j)  (in place)
 *   inv_i = rsqrt(eps + sum_j s_j^2 / hidden)
 *   y_ij  = v_ij * f32(weight[j]) * inv_i, v_ij the rounded residual (fused) or f32(input)
 *   HPRN_OUT_SAME:             out[i, j] = round_T(y_ij)      (out may be `input` itself)
 *   HPRN_OUT_FP8_E4M3_STATIC:  out[i, j] = e4m3(y_ij * (1 / *scale))
 *   HPRN_OUT_FP8_E4M3_DYNAMIC: row_scales[i] = max(max_j |y_ij|, 1e-12) / 448,
 *                              out[i, j] = e4m3(y_ij * (1 / row_scales[i]))
 * e4m3 conversion rounds to nearest even and saturates to +-448 (NaN stays NaN).
 * `input` is not written unless out == input.  `scale` (one float) and
 * `row_scales` (rows floats) are device pointers.  fp8 output needs
 * hidden % 4 == 0 with 8-byte aligned input/weight/residual rows and 4-byte
 * aligned output rows, and rows of at most 16384 vectors (262144 elements at
 * full alignment).  Output row stride is in output elements.
 */
HPRN_API int hprn_rms_norm_out(void* out, const void* input, const void* weight, void* residual,
                               int64_t rows, int64_t hidden, int64_t out_row_stride,
                               int64_t input_row_stride, int64_t residual_row_stride, double eps,
                               int dtype, int out_form, const float* scale, float* row_scales,
                               void* stream, unsigned flags);

/*
 * Gated activation (an extension past the reference):
 *   out[i, j] = round_T(act(f32(input[i, j])) * f32(input[i, d + j])),  j < d
 * Input rows hold [gate | up] (2d elements), output rows d elements; fp32
 * arithmetic with CUDA's expf / erff / tanhf.  out and input must not overlap.
 * Strides are in elements.  `act` is an hprn_act value.
 */
HPRN_API int hprn_act_and_mul(void* out, const void* input, int64_t rows, int64_t d,
                              int64_t out_row_stride, int64_t input_row_stride, int act,
                              int dtype, void* stream, unsigned flags);

/*
 * The same row operation as hprn_rms_norm_out (residual optional) with an
 * NVFP4 output (an extension past the reference): for every 16-element block
 * b of a row, with gs = *global_scale (one float on the device),
 *   block_scales[i, b] = sf = e4m3_satfinite(gs * (max_j |y_ij| / 6))
 *   q_ij = e2m1_satfinite(y_ij * (gs / sf))     (0 when sf == 0; NaN -> +6)
 * so y ~ q * sf / gs.  `out` holds two e2m1 codes per byte, element 2k in the
 * low nibble; out_row_stride counts fp4 elements (a multiple of 16).
 * block_scales is rows x hidden/16 bytes, row-major.  Needs hidden % 16 == 0,
 * 32-byte aligned input/weight/residual rows and 8-byte aligned output rows.
 */
HPRN_API int hprn_rms_norm_nvfp4(void* out, uint8_t* block_scales, const void* input,
                                 const void* weight, void* residual, int64_t rows, int64_t hidden,
                                 int64_t out_row_stride, int64_t input_row_stride,
                                 int64_t residual_row_stride, double eps, int dtype,
                                 const float* global_scale, void* stream, unsigned flags);

/*
 * The same row operation as hprn_rms_norm_out (residual optional) with a
 * per-token-group fp8 output (an extension past the reference; the
 * quantisation FP8 GEMMs with block-wise scales consume): for every group g of
 * `group_size` consecutive elements of row i,
 *   s_ig = max(max_{j in g} |y_ij|, 1e-12) / 448, rounded up to a power of two
 *          when scale_pow2 != 0 (scales an exponent-only format can hold)
 *   out[i, j] = e4m3_satfinite(y_ij * (1 / s_ig))
 *   scales[i * scale_row_stride + g * scale_group_stride] = s_ig   (fp32)
 * y_ij is the fp32 normalised value (not rounded to 16 bits first).  The
 * scale strides are in floats: (hidden / group_size, 1) for row-major scales,
 * (1, rows or more) for column-major.  group_size is 32, 64 or 128;
 * hidden % group_size == 0; input/weight/residual rows 32-byte aligned,
 * output rows 16-byte aligned; out_row_stride in bytes (fp8 elements).
 */
HPRN_API int hprn_rms_norm_fp8_group(void* out, float* scales, int64_t scale_row_stride,
                                     int64_t scale_group_stride, const void* input,
                                     const void* weight, void* residual, int64_t rows,
                                     int64_t hidden, int64_t out_row_stride,
                                     int64_t input_row_stride, int64_t residual_row_stride,
                                     double eps, int dtype, int group_size, int scale_pow2,
                                     void* stream, unsigned flags);

/*
 * Training operators (extensions past the reference).
 *
 * Workspaces: these calls allocate nothing, so a call that needs scratch
 * memory takes it from the caller.  With HPRN_WORKSPACE_QUERY in `flags` a call
 * launches nothing and writes the bytes it would need to *workspace_bytes
 * (sizes, strides and pointers as in the call to come; no tensor is read).
 * Without it, *workspace_bytes is the size of `workspace` (device memory,
 * 256-byte aligned; may be NULL when the call needs none).  The workspace is
 * free again once the call's work on the stream is done; it carries nothing
 * from one call to the next.
 */
#define HPRN_WORKSPACE_QUERY 2u

/*
 * Gated linear layer, the first half of a SwiGLU / GeGLU feed-forward block:
 *   G = input Wg^T, U = input Wu^T   (fp32 sums of 16-bit products)
 *   out[i, j] = round_T(act(G_ij) * U_ij),  j < d
 * input [rows, hidden], weight [2d, hidden] holding Wg's d rows, then Wu's.
 * gate_up (NULL, or fp32 [rows, 2d]) receives G in its first d columns and U
 * in the others, unrounded, for hprn_gated_linear_backward.  hidden == 0 gives
 * sums of nothing: 0.  Outputs must not overlap inputs or each other.
 */
HPRN_API int hprn_gated_linear(void* out, float* gate_up, const void* input, const void* weight,
                               int64_t rows, int64_t hidden, int64_t d, int64_t out_row_stride,
                               int64_t gate_up_row_stride, int64_t input_row_stride,
                               int64_t weight_row_stride, int act, int dtype, void* workspace,
                               int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Gradients of hprn_gated_linear for a gradient D of its output:
 *   S = round_T([D U act'(G) | D act(G)])
 *   grad_input [rows, hidden] = round_T(S weight)
 *   grad_weight [2d, hidden]  = round_T(S^T input)
 * gate_up: what the forward call wrote (it is not changed), or NULL to compute
 * the two products again.
 */
HPRN_API int hprn_gated_linear_backward(
    void* grad_input, void* grad_weight, const void* grad_out, const float* gate_up,
    const void* input, const void* weight, int64_t rows, int64_t hidden, int64_t d,
    int64_t grad_input_row_stride, int64_t grad_weight_row_stride, int64_t grad_out_row_stride,
    int64_t gate_up_row_stride, int64_t input_row_stride, int64_t weight_row_stride, int act,
    int dtype, void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Softmax cross entropy of a linear layer over a vocabulary, the logits never
 * held: with L = input weight^T (fp32 sums), t = target[i],
 *   lse[i]  = log sum_j exp(L_ij)
 *   loss[i] = lse[i] - L_{i, t}; 0 where t == ignore_index; NaN where t is
 *             otherwise outside [0, vocab)
 * input [rows, hidden], weight [vocab, hidden], target int64 [rows], loss and
 * lse fp32 [rows].
 */
HPRN_API int hprn_linear_cross_entropy(float* loss, float* lse, const void* input,
                                       const void* weight, const int64_t* target,
                                       int64_t ignore_index, int64_t rows, int64_t hidden,
                                       int64_t vocab, int64_t input_row_stride,
                                       int64_t weight_row_stride, int dtype, void* workspace,
                                       int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Gradients of hprn_linear_cross_entropy for gradients c[i] = grad_loss[i] of
 * the rows' losses (fp32), lse from the forward call:
 *   S_ij = c_i (exp(L_ij - lse_i) - [j == target_i]) to 16 bits; 0 in rows with
 *          target_i == ignore_index, NaN in rows with any other invalid target
 *   grad_input [rows, hidden]  = round_T(S weight)
 *   grad_weight [vocab, hidden] = round_T(S^T input)
 * S is held divided by the largest finite |c_i| (and in fp16 times 2^14), so equal
 * c_i are not all rounded alike, and in fp16 only entries below 3.7e-9 of that
 * largest one fall under the smallest normal number.  Where
 * c_i is infinite or NaN, so are row i of grad_input and grad_weight.
 */
HPRN_API int hprn_linear_cross_entropy_backward(
    void* grad_input, void* grad_weight, const float* grad_loss, const void* input,
    const void* weight, const int64_t* target, const float* lse, int64_t ignore_index,
    int64_t rows, int64_t hidden, int64_t vocab, int64_t grad_input_row_stride,
    int64_t grad_weight_row_stride, int64_t input_row_stride, int64_t weight_row_stride, int dtype,
    void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Gradients of RMSNorm, y = x w inv, inv = rsqrt(mean(x^2) + eps), for a
 * gradient D of y:
 *   grad_input  = round_T(inv (w D - x inv mean(w D x inv)) + grad_residual)
 *   grad_weight = round_T(sum over rows of D x inv)
 * For the fused add + RMSNorm `input` is the updated residual, and grad_input
 * the gradient of both its addends.  grad_residual (NULL for none): the
 * gradient that reaches `input` through the residual branch.
 */
HPRN_API int hprn_rms_norm_backward(void* grad_input, void* grad_weight, const void* grad_out,
                                    const void* input, const void* weight,
                                    const void* grad_residual, int64_t rows, int64_t hidden,
                                    int64_t grad_input_row_stride, int64_t grad_out_row_stride,
                                    int64_t input_row_stride, int64_t grad_residual_row_stride,
                                    double eps, int dtype, void* workspace,
                                    int64_t* workspace_bytes, void* stream, unsigned flags);

/* One gradient tensor of hprn_grad_norm / hprn_grad_clip: rows x cols elements
 * of an hprn_dtype; `out` is read by hprn_grad_clip only. */
typedef struct hprn_grad {
  const void* grad;
  void* out;
  int64_t rows, cols;
  int64_t row_stride, out_row_stride;
  int32_t dtype, out_dtype;
} hprn_grad;

/*
 * *norm = sqrt(sum of the squares of all elements of all tensors) (fp32 on the
 * device; 0 for no elements).  `grads` is a host array, read during the call.
 * The same tensors give the same bits on every call.
 */
HPRN_API int hprn_grad_norm(float* norm, const hprn_grad* grads, int64_t count, void* workspace,
                            int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * out = round(grad * min(1, max_norm / (*norm + 1e-6))) for every tensor; a NaN
 * norm makes every output NaN.  `out` may be the gradient itself (same type and
 * stride), which is then left unwritten where the factor is 1; otherwise it must not overlap it.
 * No `out` may share elements with another tensor of the list or with `norm` (not checked:
 * rows of several tensors may lie interleaved); a tensor listed twice is one such.
 */
HPRN_API int hprn_grad_clip(const hprn_grad* grads, int64_t count, const float* norm,
                            double max_norm, void* stream, unsigned flags);

/*
 * hprn_grad_norm and hprn_grad_clip in one call, the same results.
 */
HPRN_API int hprn_clip_grad_norm(float* norm, const hprn_grad* grads, int64_t count,
                                 double max_norm, void* workspace, int64_t* workspace_bytes,
                                 void* stream, unsigned flags);

/*
 * The norms before and after a gated block in one pass (extension):
 *   y   = input inv_x post_weight, inv_x = rsqrt(eps + mean(input^2))
 *         (y = input where post_weight is NULL)
 *   t   = residual_scale residual + gate y       (fp32; residual_out = round_T(t))
 *   out = round_T(t inv_t weight), inv_t = rsqrt(eps + mean(t^2))  (t unrounded)
 * input is a block's output, out what the next block reads.  gate: NULL (1), or
 * rows / rows_per_gate rows of gate_width values, gate_width 1 or hidden; gate
 * row k serves rows k rows_per_gate to (k + 1) rows_per_gate - 1.  out may be
 * input, and residual_out residual, with the same stride; outputs must not
 * otherwise overlap anything.
 */
HPRN_API int hprn_gated_add_rms_norm(void* out, void* residual_out, const void* input,
                                     const void* residual, const void* post_weight,
                                     const void* weight, const void* gate, int64_t rows,
                                     int64_t hidden, int64_t rows_per_gate, int64_t gate_width,
                                     int64_t out_row_stride, int64_t residual_out_row_stride,
                                     int64_t input_row_stride, int64_t residual_row_stride,
                                     int64_t gate_row_stride, double residual_scale, double eps,
                                     int dtype, void* stream, unsigned flags);

/*
 * Gradients of hprn_gated_add_rms_norm for gradients D of out and E
 * (grad_residual_out; NULL for none) of residual_out.  residual_out is what the
 * forward call wrote.  With n = residual_out inv_t, m = input inv_x (m = input,
 * post_weight = 1 where that is NULL), g the gate, means over a row:
 *   dt = inv_t (weight D - n mean(weight D n)) + E
 *   grad_residual    = round_T(residual_scale dt)
 *   grad_gate        = round_T(sum of dt m post_weight over what shares a value)
 *   grad_input       = round_T(inv_x (g post_weight dt - m mean(g post_weight dt m)))
 *                      (round_T(g dt) without post_weight)
 *   grad_post_weight = round_T(sum over rows of g dt m)    (not without post_weight)
 *   grad_weight      = round_T(sum over rows of D n)
 * grad_gate has the gate's rows and width.
 */
HPRN_API int hprn_gated_add_rms_norm_backward(
    void* grad_input, void* grad_residual, void* grad_post_weight, void* grad_weight,
    void* grad_gate, const void* grad_out, const void* grad_residual_out, const void* input,
    const void* residual_out, const void* post_weight, const void* weight, const void* gate,
    int64_t rows, int64_t hidden, int64_t rows_per_gate, int64_t gate_width,
    int64_t grad_input_row_stride, int64_t grad_residual_row_stride, int64_t grad_gate_row_stride,
    int64_t grad_out_row_stride, int64_t grad_residual_out_row_stride, int64_t input_row_stride,
    int64_t residual_out_row_stride, int64_t gate_row_stride, double residual_scale, double eps,
    int dtype, void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Log probabilities under the softmax of a linear layer over a vocabulary
 * (extension): with L = input weight^T / temperature (fp32 sums), t = target[i],
 *   lse[i]      = log sum_j exp(L_ij)
 *   log_prob[i] = L_{i, t} - lse[i]; 0 where t == ignore_index; NaN where t is
 *                 otherwise outside [0, vocab)
 *   entropy[i]  = -sum_j p_ij log p_ij, p_ij = exp(L_ij - lse[i]); 0 where
 *                 t == ignore_index
 *   top_log_probs[i, k], top_indices[i, k], k < top: the largest L_ij - lse[i] of
 *                 every row, the largest first, and their j.  They are ordered by
 *                 logits summed in 64 bits, equal ones by their indices; a logit
 *                 is missed only where more than four others lie between it and
 *                 the last place within the rounding of an fp32 sum.  In rows with a
 *                 NaN logit the values are NaN and the indices any.
 * 1e-30 <= temperature <= 1e30; 0 <= top <= 64, top <= vocab; top_* may be NULL
 * where top is 0.  The outputs of
 * rows are dense.  With top > 0 the workspace holds the logits of a block of rows,
 * 1 GiB at most where 256 rows fit in that.
 */
HPRN_API int hprn_linear_log_probs(float* log_prob, float* entropy, float* lse,
                                   float* top_log_probs, int64_t* top_indices, const void* input,
                                   const void* weight, const int64_t* target, int64_t ignore_index,
                                   double temperature, int64_t top, int64_t rows, int64_t hidden,
                                   int64_t vocab, int64_t input_row_stride,
                                   int64_t weight_row_stride, int dtype, void* workspace,
                                   int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Gradients of hprn_linear_log_probs for gradients g of log_prob and h of entropy
 * (fp32; grad_entropy NULL for none, entropy is then not read); lse and entropy
 * from the forward call:
 *   S_ij = (g_i ([j == t_i] - p_ij) - h_i p_ij (log p_ij + entropy_i)) / temperature
 *          to 16 bits; 0 in rows with target_i == ignore_index, NaN in rows with any
 *          other invalid target
 *   grad_input [rows, hidden]   = round_T(S weight)
 *   grad_weight [vocab, hidden] = round_T(S^T input)
 * S is held divided by the largest finite |g_i| or |h_i| (and in fp16 times 2^14, or
 * 2^13 with grad_entropy).  Where g_i or h_i is infinite or NaN, so are row i of
 * grad_input and grad_weight.
 */
HPRN_API int hprn_linear_log_probs_backward(
    void* grad_input, void* grad_weight, const float* grad_log_prob, const float* grad_entropy,
    const void* input, const void* weight, const int64_t* target, const float* lse,
    const float* entropy, int64_t ignore_index, double temperature, int64_t rows, int64_t hidden,
    int64_t vocab, int64_t grad_input_row_stride, int64_t grad_weight_row_stride,
    int64_t input_row_stride, int64_t weight_row_stride, int dtype, void* workspace,
    int64_t* workspace_bytes, void* stream, unsigned flags);

/*
 * Rows quantised to 8-bit integers with one scale each (extension):
 *   t = input, or input + residual (fp32; residual_out = round_T of it)
 *   y = t weight rsqrt(eps + mean(t^2)), or y = t where weight is NULL
 *   scales[i] = max(max_j |y_ij|, 1e-12) / 127,  out_ij = round(y_ij (1 / scales[i])),
 * to nearest even, in [-127, 127]; t is not rounded in between; hidden >= 1.  residual and
 * residual_out go together and may be one tensor; a row with a NaN has a NaN scale,
 * one with an infinity an infinite or NaN scale.
 */
HPRN_API int hprn_rms_norm_int8(int8_t* out, float* scales, void* residual_out, const void* input,
                                const void* weight, const void* residual, int64_t rows,
                                int64_t hidden, int64_t out_row_stride,
                                int64_t residual_out_row_stride, int64_t input_row_stride,
                                int64_t residual_row_stride, double eps, int dtype, void* stream,
                                unsigned flags);

/*
 * Linear layer in 8-bit integers (extension):
 *   out_ij = round_T(S_ij input_scale[i] weight_scale[j] + bias[j]),
 *   S_ij = sum_k input_ik weight_jk, exact in 32 bits (hidden <= 131071) and
 * rounded to fp32 once.  input int8 [rows, hidden], weight int8 [channels, hidden],
 * scales fp32, bias (NULL for none) and out of type `dtype`.  Rows of an even
 * length on 16-byte boundaries are read as they are, others are copied first.
 */
HPRN_API int hprn_linear_int8(void* out, const int8_t* input, const float* input_scale,
                              const int8_t* weight, const float* weight_scale, const void* bias,
                              int64_t rows, int64_t hidden, int64_t channels,
                              int64_t out_row_stride, int64_t input_row_stride,
                              int64_t weight_row_stride, int dtype, void* workspace,
                              int64_t* workspace_bytes, void* stream, unsigned flags);

/* Message for the last non-OK status returned on this thread ("" if none). */
HPRN_API const char* hprn_last_error(void);

/* Static name of a status code. */
HPRN_API const char* hprn_status_string(int status);

/* HPRN_VERSION of the loaded library. */
HPRN_API int hprn_version(void);

/*
 * Launch-plan introspection (for tests and benchmarks): writes the plan that
 * hprn_rms_norm would use for this problem on the current device into
 * `plan` as a NUL-terminated string "<kind>:vec<V>:vpt<P>:tpr<T>:cluster<C>:rpc<R>"
 * (kind warp | cta | cluster | twopass | tma; V bytes per vector access; P
 * vectors per thread; T threads per CTA, or for kind warp the lanes holding one
 * row (1..32, a power of two); C CTAs per row; R rows per CTA, or for kind tma
 * the depth of the CTA's ring of TMA-staged rows) and returns HPRN_OK.  Performs no launch.  Null input/residual pointers plan for
 * 256-byte-aligned tensors; without a usable device it plans for a 148-SM B200.
 * The weight is assumed to be aligned like the input: a call whose weight is
 * less aligned than its input gets a narrower vector width (and so possibly
 * another plan) than the one returned here.
 */
HPRN_API int hprn_rms_norm_plan(int64_t rows, int64_t hidden, int dtype, const void* input,
                                const void* residual, int64_t input_row_stride,
                                int64_t residual_row_stride, char* plan, int plan_len);

/*
 * Tuning hook: force the launch plan of every later hprn_rms_norm* call in
 * this process (same string format as hprn_rms_norm_plan; NULL or "" restores
 * the built-in heuristic).  A plan may end in ":pf<F>:et<E>", two launch knobs
 * that change timing only, never results: F is the L2 prefetch each CTA issues
 * for its first rows before waiting on the preceding grid (0 none, 1 the
 * grid's first wave of CTAs, 2 every CTA, 3 the first wave, with every CTA also
 * prefetching the row of the CTA one wave later) and E where dependents are triggered
 * (0 after the last store, 1 after the row reduction, 2 once the loads are
 * issued); without them the plan's defaults apply.  "default:pf<F>:et<E>" keeps the built-in plan and sets only
 * the knobs.  hprn_rms_norm_plan echoes knobs an override names.  The
 * HP_RMS_NORM_PLAN environment variable, read at
 * the first call, sets the same override.  A forced plan that does not fit a
 * call makes that call fail with HPRN_ERR_INVALID_ARGUMENT.  Process-global
 * (safe to call concurrently with launches): meant for benchmarks and
 * launch-shape sweeps, not for production callers.
 */
HPRN_API int hprn_set_plan_override(const char* plan);

/*
 * No reference counterpart.  Kernels that wait on mbarriers for asynchronous
 * copies and matrix instructions do so with a bound (one second): those that
 * stage rows of hprn_rms_norm* through TMA bulk copies (plan kind tma, reached
 * only through a plan override), the matrix products of hprn_gated_linear*,
 * hprn_linear_cross_entropy*, hprn_linear_log_probs* and hprn_linear_int8, and
 * hprn_rms_norm_backward and hprn_gated_add_rms_norm_backward.  A CTA that gives up
 * a wait stops, once its copies in flight have landed, and counts itself here,
 * on its device: in the tma plans it leaves the row it gave up on and its
 * remaining rows untouched (input and residual as they were), in the others
 * the outputs it had not written.  The call that launched it still returns
 * HPRN_OK; later calls of these operators on that device return HPRN_ERR_CUDA once a launch of
 * these has given up a wait, until the count is reset.  No wait gives up on a
 * GPU that works.
 * Writes the current device's count into *count and, if `reset` is non-zero,
 * clears it.  Synchronous; synchronise the streams that launched the kernels
 * first.  A non-zero count means the launches since the last reset produced
 * incomplete results.
 */
HPRN_API int hprn_wait_timeouts(unsigned int* count, int reset);

/*
 * No reference counterpart.  Test hook for the bounded waits above: every
 * later launch of a TMA-staged plan in this process makes the staged copy of
 * row `row` (counted from the first row of that call; -1 turns the hook off)
 * expect 16 bytes more than its copies deliver, so the row's mbarrier phase
 * cannot complete and its wait runs out after `wait_limit_ns` nanoseconds
 * (at most one second; 0 keeps the built-in one second).  The CTA holding
 * that row then takes its give-up path: it waits for the copies it still has
 * in flight (releasing the stalled row's 16 extra bytes itself, so that wait
 * ends once its copies have landed), leaves that row and its later rows
 * untouched, and counts itself in hprn_wait_timeouts.  No fault and no hang:
 * every wait stays bounded.  Plans of other kinds ignore it.  Process-global;
 * for tests only.
 */
HPRN_API int hprn_test_stall_bulk_copy(int64_t row, uint64_t wait_limit_ns);

/*
 * No reference counterpart.  Test hook for the same waits of the training
 * operators: while `on` is non-zero, every launch of their matrix products and
 * of the norms' backward kernels loads nothing, so that its waits run out, after
 * `wait_limit_ns` nanoseconds each (at most one second; 0 keeps that), and its
 * CTAs take their give-up path.  No fault and no hang: every wait stays
 * bounded.  Process-global; for tests only.
 */
HPRN_API int hprn_test_stall_loads(int on, uint64_t wait_limit_ns);

/*
 * No reference counterpart.  Test hook, launches nothing: how
 * hprn_linear_cross_entropy_backward takes the input gradient's sums over piece
 * `piece` of the vocabulary.  Writes to out[0..3] the number of pieces, the
 * piece's columns, the stages of 64 terms that these make, and the shares that
 * the stages are dealt out to.
 */
HPRN_API int hprn_test_loss_backward_piece(int64_t rows, int64_t hidden, int64_t vocab,
                                           int64_t piece, int64_t* out);

/*
 * No reference counterpart.  Test hook, launches and reads nothing: what the row
 * kernels of hprn_gated_add_rms_norm and hprn_rms_norm_int8 read of a tensor whose
 * rows lie off 16-byte boundaries, `start` elements behind one.  Writes to out[0..2]
 * the most elements read before the tensor, the most behind it, and the vectors of
 * which an element is not read.
 */
HPRN_API int hprn_test_loose_reads(int64_t rows, int64_t hidden, int64_t row_stride, int64_t start,
                                   int64_t* out);

#ifdef __cplusplus
}
#endif

#endif /* HP_RMS_NORM_B200_H_ */
