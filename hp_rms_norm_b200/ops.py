"""Python API.

The reference's two functions, argument for argument (hp_rms_norm/ops.py:4-24):
``hp_rms_norm(input, weight, residual, eps)`` runs the fused residual add +
RMSNorm in place (``residual += input``; ``input = RMSNorm(residual) * weight``)
and returns None; ``relu(output, input)`` writes ``torch.relu(input)`` into
``output`` and returns None.

Extensions (not in the reference): ``rms_norm`` (plain RMSNorm),
``fused_add_rms_norm`` (the fused op into a separate output) and
``rms_norm_fp8`` (either form with an fp8 e4m3 output, static or per-row
scale), ``rms_norm_nvfp4`` (NVFP4 output), and the gated activations ``silu_and_mul``, ``gelu_and_mul`` and
``gelu_tanh_and_mul``; ``gated_add_rms_norm`` (the norms on both sides of a gated block) and its
backward pass; ``linear_log_probs`` (log probabilities of given tokens, entropy and best
alternatives) and its backward pass; ``rms_norm_int8``, ``quantize_int8`` and ``linear_int8``
(products of 8-bit integers and what feeds them); and for training ``gated_linear`` (a feed-forward block's gate and up
products with the activation), ``linear_cross_entropy`` (the loss of a linear layer over a
vocabulary, without its logits), their backward passes, ``rms_norm_backward``, and
``grad_norm`` / ``clip_grad_norm``.  Everything dispatches through ``torch.ops.hp_rms_norm``, registered
by this package's compiled ``_C`` extension.
"""
from typing import NamedTuple, Optional

import torch

_ops = torch.ops.hp_rms_norm


def hp_rms_norm(
    input,
    weight,
    residual,
    eps,
):
    torch.ops.hp_rms_norm.rms_norm.default(input, weight, residual, eps)


def relu(
    output,
    input,
):
    torch.ops.hp_rms_norm.relu.default(output, input)


def rms_norm(input, weight, eps, out=None):
    """RMSNorm without a residual: out = input * rsqrt(mean(input^2) + eps) * weight,
    in the input's dtype; ``out`` may be ``input`` (in place).  Returns ``out``."""
    if out is None:
        out = torch.empty_like(input)
    torch.ops.hp_rms_norm.rms_norm_out.default(out, input, weight, None, eps)
    return out


def fused_add_rms_norm(input, residual, weight, eps, out=None):
    """``hp_rms_norm`` into a separate output: residual += input (in place);
    out = RMSNorm(residual) * weight; ``input`` is left unchanged unless it is
    ``out``.  Returns ``out``."""
    if out is None:
        out = torch.empty_like(input)
    torch.ops.hp_rms_norm.rms_norm_out.default(out, input, weight, residual, eps)
    return out


def rms_norm_fp8(input, weight, eps, residual=None, scale=None, out=None):
    """RMSNorm (fused with ``residual += input`` when a residual is given) with
    an fp8 e4m3 output.  With ``scale`` (a one-element float32 tensor) the output
    is e4m3(y / scale); without it, each row gets scale max|y| / 448, returned
    as a float32 tensor of shape input.shape[:-1].  Returns (out, scales)."""
    if out is None:
        out = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    if scale is not None:
        torch.ops.hp_rms_norm.rms_norm_fp8.default(out, input, weight, residual, eps, scale, None)
        return out, scale
    row_scales = torch.empty(input.shape[:-1], dtype=torch.float32, device=input.device)
    torch.ops.hp_rms_norm.rms_norm_fp8.default(out, input, weight, residual, eps, None, row_scales)
    return out, row_scales


def rms_norm_nvfp4(input, weight, eps, global_scale, residual=None):
    """RMSNorm (fused with ``residual += input`` when a residual is given) with
    an NVFP4 output: returns (codes, block_scales), codes uint8
    [..., hidden/2] holding two e2m1 values per byte (element 2k in the low
    nibble), block_scales float8_e4m3fn [..., hidden/16]; the normalised value
    is approximately e2m1 * block_scale / global_scale (``global_scale`` a
    one-element float32 tensor)."""
    h = input.shape[-1]
    codes = torch.empty(input.shape[:-1] + (h // 2,), dtype=torch.uint8, device=input.device)
    scales = torch.empty(input.shape[:-1] + (h // 16,), dtype=torch.float8_e4m3fn,
                         device=input.device)
    torch.ops.hp_rms_norm.rms_norm_nvfp4.default(codes, scales, input, weight, residual, eps,
                                                 global_scale)
    return codes, scales


def rms_norm_fp8_group(input, weight, eps, residual=None, group_size=128, scale_pow2=False,
                       column_major_scales=False):
    """RMSNorm (fused with ``residual += input`` when a residual is given) with a
    per-token-group fp8 output: returns (out, scales), out float8_e4m3fn
    [..., hidden], scales float32 [rows, hidden / group_size] (rows = the
    leading dimensions flattened) with out ~ y / scale per group of
    ``group_size`` elements.  ``scale_pow2`` rounds scales up to powers of two;
    ``column_major_scales`` returns a transposed view of a [hidden /
    group_size, rows] buffer (the layout block-scaled FP8 GEMMs read)."""
    h = input.shape[-1]
    rows = input.numel() // h if h else 0
    out = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    if column_major_scales:
        scales = torch.empty((h // group_size, rows), dtype=torch.float32, device=input.device).t()
    else:
        scales = torch.empty((rows, h // group_size), dtype=torch.float32, device=input.device)
    torch.ops.hp_rms_norm.rms_norm_fp8_group.default(out, scales, input, weight, residual, eps,
                                                     group_size, scale_pow2)
    return out, scales


def _act_and_mul(op, input, out):
    if out is None:
        out = torch.empty(input.shape[:-1] + (input.shape[-1] // 2,), dtype=input.dtype,
                          device=input.device)
    op(out, input)
    return out


def silu_and_mul(input, out=None):
    """out = silu(input[..., :d]) * input[..., d:], d = input.shape[-1] // 2."""
    return _act_and_mul(torch.ops.hp_rms_norm.silu_and_mul.default, input, out)


def gelu_and_mul(input, out=None):
    """out = gelu(input[..., :d]) * input[..., d:] (erf form)."""
    return _act_and_mul(torch.ops.hp_rms_norm.gelu_and_mul.default, input, out)


def gelu_tanh_and_mul(input, out=None):
    """out = gelu_tanh(input[..., :d]) * input[..., d:] (tanh approximation)."""
    return _act_and_mul(torch.ops.hp_rms_norm.gelu_tanh_and_mul.default, input, out)


def _new_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def gated_linear(input, weight, act="silu", out=None, gate_up=None):
    """out = act(input Wg^T) * (input Wu^T), the first half of a SwiGLU / GeGLU feed-forward
    block in one kernel.  ``input`` [..., hidden], ``weight`` [2 d, hidden] holding Wg's rows,
    then Wu's (the order ``silu_and_mul`` reads its halves in); ``act`` 'silu', 'gelu' or
    'gelu_tanh'.  ``gate_up``, a float32 [..., 2 d] tensor, receives the two products for
    ``gated_linear_backward``.  Returns ``out`` [..., d]."""
    if out is None:
        out = input.new_empty(input.shape[:-1] + (weight.shape[0] // 2,))
    _ops.gated_linear.default(out, gate_up, input, weight, act)
    return out


def gated_linear_backward(grad_out, input, weight, act="silu", gate_up=None):
    """Gradients (grad_input, grad_weight) of ``gated_linear`` for a gradient of its output.
    With the ``gate_up`` that the forward call wrote the two products are read from it, without
    it they are computed again."""
    grad_input = _new_like(input)
    grad_weight = _new_like(weight)
    _ops.gated_linear_backward.default(grad_input, grad_weight, grad_out, input,
                                                        weight, gate_up, act)
    return grad_input, grad_weight


def linear_cross_entropy(input, weight, target, ignore_index=-100):
    """Per-row cross entropy of softmax(input weight^T) against ``target``, without holding the
    logits: ``input`` [..., hidden], ``weight`` [vocab, hidden], ``target`` int64 [...].
    Returns (loss, lse), float32 [...]: the loss (0 where the target is ``ignore_index``, NaN
    where it is otherwise outside the vocabulary) and the logits' log-sum-exp, which
    ``linear_cross_entropy_backward`` takes."""
    loss = torch.empty(input.shape[:-1], dtype=torch.float32, device=input.device)
    lse = torch.empty_like(loss)
    _ops.linear_cross_entropy.default(loss, lse, input, weight, target,
                                                       ignore_index)
    return loss, lse


def linear_cross_entropy_backward(grad_loss, input, weight, target, lse, ignore_index=-100):
    """Gradients (grad_input, grad_weight) of ``linear_cross_entropy`` for the gradients of the
    rows' losses, ``grad_loss`` float32 [...]; the logits are computed again, one piece of the
    vocabulary at a time."""
    grad_input = _new_like(input)
    grad_weight = _new_like(weight)
    _ops.linear_cross_entropy_backward.default(
        grad_input, grad_weight, grad_loss, input, weight, target, lse, ignore_index)
    return grad_input, grad_weight


def rms_norm_backward(grad_out, input, weight, eps, grad_residual=None):
    """Gradients (grad_input, grad_weight) of RMSNorm for a gradient of its output.  For the
    fused forms ``input`` is the updated residual, and ``grad_residual`` the gradient that
    reaches it from its other uses, which is added: grad_input is then the gradient of both
    addends."""
    grad_input = _new_like(input)
    grad_weight = _new_like(weight)
    _ops.rms_norm_backward.default(grad_input, grad_weight, grad_out, input,
                                                    weight, grad_residual, eps)
    return grad_input, grad_weight


def grad_norm(grads):
    """The 2-norm over all elements of all tensors of ``grads`` (float32, bfloat16 or float16,
    mixed as they come), a float32 scalar tensor."""
    if not len(grads):
        return torch.zeros((), dtype=torch.float32)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    _ops.grad_norm.default(norm, grads)
    return norm


def clip_grad_norm(grads, max_norm, out=None):
    """Scales every gradient by min(1, max_norm / (norm + 1e-6)), norm the 2-norm over all of
    them, in place or into the tensors of ``out`` (of any of the three types: 16-bit gradients
    into an optimiser's float32 buffers, say).  What is written may share elements with no
    other tensor of the call, so a tensor is listed once.  Returns the norm before clipping, a
    float32 scalar tensor; nothing waits for the GPU."""
    if not len(grads):
        return torch.zeros((), dtype=torch.float32)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    _ops.clip_grad_norm.default(grads if out is None else out, norm, grads, max_norm)
    return norm


def gated_add_rms_norm(input, residual, post_weight, weight, eps, gate=None, residual_scale=1.0,
                       out=None, residual_out=None):
    """The end of one block and the norm before the next in one pass:

        residual_out = residual_scale * residual + gate * (RMSNorm(input) * post_weight)
        out = RMSNorm(residual_out) * weight

    ``residual_out`` None updates ``residual`` in place.  ``post_weight`` None leaves the norm after
    the block out.  ``gate`` None is 1; otherwise its shape is one that broadcasts over
    ``input``'s trailing leading dimensions: [hidden] (a learned gate for each channel), [batch, 1,
    hidden] (one for each sequence), input's own shape, or any of these with a last dimension
    of 1.  The sums are fp32 and ``out`` comes from the unrounded new residual.  Returns ``out``."""
    if out is None:
        out = torch.empty_like(input)
    if residual_out is None or residual_out is residual:
        _ops.gated_add_rms_norm.default(out, residual, None, input, post_weight, weight, gate,
                                        residual_scale, eps)
    else:
        _ops.gated_add_rms_norm_sum.default(out, residual_out, input, residual, post_weight, weight,
                                            gate, residual_scale, eps)
    return out


def gated_add_rms_norm_backward(grad_out, input, residual, post_weight, weight, eps, gate=None,
                                residual_scale=1.0, grad_residual=None):
    """Gradients (grad_input, grad_residual, grad_post_weight, grad_weight, grad_gate) of
    ``gated_add_rms_norm`` for a gradient of ``out`` and, with ``grad_residual``, one that reaches
    the new residual from its other uses.  ``residual`` is the new residual that the forward call
    wrote.  grad_post_weight and grad_gate are None where their tensors are."""
    grad_input, grad_old, grad_post, grad_weight, grad_gate = _ops.gated_add_rms_norm_backward.default(
        grad_out, grad_residual, input, residual, post_weight, weight, gate, residual_scale, eps)
    return (grad_input, grad_old, None if post_weight is None else grad_post, grad_weight,
            None if gate is None else grad_gate)


class LogProbs(NamedTuple):
    """What ``linear_log_probs`` returns; the last two are None without ``top``."""
    log_prob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_log_probs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def linear_log_probs(input, weight, target, top=0, temperature=1.0, ignore_index=-100):
    """Log probabilities under softmax(input weight^T / temperature) without holding the logits:
    ``input`` [..., hidden], ``weight`` [vocab, hidden], ``target`` int64 [...].  Returns a
    ``LogProbs``: log_prob and entropy, float32 [...] (0 where the target is ``ignore_index``; the
    log probability of any other target outside the vocabulary is NaN), lse, the log-sum-exp
    that ``linear_log_probs_backward`` takes, and for ``top`` > 0 (at most 64) the largest log
    probabilities of every row, float32 [..., top], with their int64 indices: the largest first,
    equal ones by their indices."""
    log_prob, entropy, lse, values, indices = _ops.linear_log_probs.default(
        input, weight, target, top, temperature, ignore_index)
    return LogProbs(log_prob, entropy, lse, values if top else None, indices if top else None)


def linear_log_probs_backward(grad_log_prob, input, weight, target, lse, entropy=None,
                              grad_entropy=None, temperature=1.0, ignore_index=-100):
    """Gradients (grad_input, grad_weight) of ``linear_log_probs`` for gradients of the rows' log
    probabilities and, where ``grad_entropy`` is given (with the forward call's ``entropy``), of
    their entropies, float32 [...]; the logits are computed again, one piece of the vocabulary at
    a time."""
    return _ops.linear_log_probs_backward.default(grad_log_prob, grad_entropy, input, weight, target, lse,
                                                  entropy, temperature, ignore_index)


def rms_norm_int8(input, weight, eps, residual=None, residual_out=None):
    """RMSNorm (with a residual: of residual + input, which goes to ``residual_out``, or to
    ``residual`` itself without one) with an int8 output and one scale a row: returns (codes,
    scales), codes int8 of input's shape, scales float32 [...] = max|y| / 127, y ~ codes *
    scale.  ``linear_int8`` takes both."""
    if residual is None or residual_out is None or residual_out is residual:
        return _ops.rms_norm_int8.default(input, weight, residual, residual_out, eps)
    return _ops.rms_norm_int8_sum.default(input, weight, residual, residual_out, eps)


def quantize_int8(input):
    """``input`` itself as int8 codes with one scale a row: (codes, scales) as ``rms_norm_int8``."""
    return rms_norm_int8(input, None, 0.0)


def linear_int8(input, input_scale, weight, weight_scale, bias=None, dtype=torch.bfloat16, out=None):
    """out = (input weight^T) * input_scale * weight_scale + bias in 8-bit integers: ``input`` int8
    [..., hidden] with a float32 scale for each row (``rms_norm_int8``, ``quantize_int8``),
    ``weight`` int8 [channels, hidden] with a float32 scale for each channel, ``bias`` [channels]
    of type ``dtype`` (bfloat16 or float16).  The sums are exact.  Returns ``out`` [..., channels]
    of type ``dtype``."""
    if out is None:
        return _ops.linear_int8.default(input, input_scale, weight, weight_scale, bias, dtype)
    _ops.linear_int8.out(out, input, input_scale, weight, weight_scale, bias)
    return out


__all__ = ["hp_rms_norm", "relu", "rms_norm", "fused_add_rms_norm", "rms_norm_fp8", "rms_norm_nvfp4",
           "rms_norm_fp8_group", "silu_and_mul", "gelu_and_mul", "gelu_tanh_and_mul",
           "gated_linear", "gated_linear_backward", "linear_cross_entropy",
           "linear_cross_entropy_backward", "rms_norm_backward", "grad_norm", "clip_grad_norm",
           "gated_add_rms_norm", "gated_add_rms_norm_backward", "LogProbs", "linear_log_probs",
           "linear_log_probs_backward", "rms_norm_int8", "quantize_int8", "linear_int8", "torch"]
