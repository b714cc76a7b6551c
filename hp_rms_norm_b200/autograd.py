"""The operators that have a backward pass, as torch.autograd functions.

``rms_norm``, ``fused_add_rms_norm``, ``gated_add_rms_norm``, ``gated_linear``,
``linear_cross_entropy`` and ``linear_log_probs`` take and return tensors like torch's own functions do;
their forward and backward passes are the kernels behind the functions of
``hp_rms_norm_b200.ops`` with the same names.  Nothing is changed in place: the
values a backward pass needs (a block's residual among them) stay as they were.
The gradients have no gradients of their own: a second derivative is refused.
"""
import torch
from torch.autograd.function import once_differentiable

from . import ops


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, eps):
        ctx.save_for_backward(input, weight)
        ctx.eps = eps
        return ops.rms_norm(input, weight, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        input, weight = ctx.saved_tensors
        grad_input, grad_weight = ops.rms_norm_backward(grad_out.contiguous(), input, weight, ctx.eps)
        return grad_input, grad_weight, None


class _FusedAddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, residual, weight, eps):
        total = residual.clone(memory_format=torch.contiguous_format)
        out = ops.fused_add_rms_norm(input, total, weight, eps)
        ctx.save_for_backward(total, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)  # a last block's sum has no user, so no gradient to read
        return out, total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_total):
        if grad_out is None:
            return grad_total, grad_total, None, None
        total, weight = ctx.saved_tensors
        if grad_total is not None:
            grad_total = grad_total.contiguous()
        grad, grad_weight = ops.rms_norm_backward(grad_out.contiguous(), total, weight, ctx.eps,
                                                  grad_residual=grad_total)
        return grad, grad, grad_weight, None


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, act, keep_products):
        gate_up = None
        if keep_products and any(ctx.needs_input_grad[:2]):
            gate_up = torch.empty(input.shape[:-1] + weight.shape[:1], dtype=torch.float32,
                                  device=input.device)
        out = ops.gated_linear(input, weight, act, gate_up=gate_up)
        ctx.save_for_backward(input, weight, gate_up)
        ctx.act = act
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        input, weight, gate_up = ctx.saved_tensors
        grad_input, grad_weight = ops.gated_linear_backward(grad_out.contiguous(), input, weight,
                                                            ctx.act, gate_up=gate_up)
        return grad_input, grad_weight, None, None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, target, ignore_index):
        loss, lse = ops.linear_cross_entropy(input, weight, target, ignore_index)
        ctx.save_for_backward(input, weight, target, lse)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        input, weight, target, lse = ctx.saved_tensors
        grad_input, grad_weight = ops.linear_cross_entropy_backward(
            grad_loss.contiguous(), input, weight, target, lse, ctx.ignore_index)
        return grad_input, grad_weight, None, None


class _GatedAddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, residual, post_weight, weight, gate, eps, residual_scale):
        total = torch.empty_like(residual, memory_format=torch.contiguous_format)
        out = ops.gated_add_rms_norm(input, residual, post_weight, weight, eps, gate=gate,
                                     residual_scale=residual_scale, residual_out=total)
        ctx.save_for_backward(input, total, post_weight, weight, gate)
        ctx.eps, ctx.residual_scale = eps, residual_scale
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_total):
        input, total, post_weight, weight, gate = ctx.saved_tensors
        if grad_out is None:
            if grad_total is None:
                return (None,) * 7
            grad_out = torch.zeros_like(total)
        if grad_total is not None:
            grad_total = grad_total.contiguous()
        grads = ops.gated_add_rms_norm_backward(grad_out.contiguous(), input, total, post_weight,
                                                weight, ctx.eps, gate=gate,
                                                residual_scale=ctx.residual_scale,
                                                grad_residual=grad_total)
        return grads + (None, None)


class _LinearLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, target, temperature, ignore_index):
        found = ops.linear_log_probs(input, weight, target, temperature=temperature,
                                     ignore_index=ignore_index)
        ctx.save_for_backward(input, weight, target, found.lse, found.entropy)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.set_materialize_grads(False)
        return found.log_prob, found.entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_log_prob, grad_entropy):
        if grad_log_prob is None and grad_entropy is None:
            return (None,) * 5
        input, weight, target, lse, entropy = ctx.saved_tensors
        if grad_log_prob is None:
            grad_log_prob = torch.zeros_like(grad_entropy)
        if grad_entropy is not None:
            grad_entropy = grad_entropy.contiguous()
        grad_input, grad_weight = ops.linear_log_probs_backward(
            grad_log_prob.contiguous(), input, weight, target, lse, entropy=entropy,
            grad_entropy=grad_entropy, temperature=ctx.temperature, ignore_index=ctx.ignore_index)
        return grad_input, grad_weight, None, None, None


def rms_norm(input, weight, eps):
    """RMSNorm(input) * weight."""
    return _RMSNorm.apply(input, weight, eps)


def fused_add_rms_norm(input, residual, weight, eps):
    """(RMSNorm(total) * weight, total) for total = input + residual."""
    return _FusedAddRMSNorm.apply(input, residual, weight, eps)


def gated_add_rms_norm(input, residual, post_weight, weight, eps, gate=None, residual_scale=1.0):
    """(RMSNorm(total) * weight, total) for total = residual_scale * residual + gate *
    (RMSNorm(input) * post_weight); ``post_weight`` and ``gate`` as in ``ops.gated_add_rms_norm``."""
    return _GatedAddRMSNorm.apply(input, residual, post_weight, weight, gate, eps, residual_scale)


def gated_linear(input, weight, act="silu", keep_products=True):
    """act(input Wg^T) * (input Wu^T), ``weight`` = [Wg; Wu].  ``keep_products`` keeps the two
    products (float32, 8 bytes for each output element) for the backward pass; without it they
    are computed again there.  Where no graph is recorded nothing is kept."""
    # needs_input_grad tells a leaf's wish, not whether a graph is being recorded.
    return _GatedLinear.apply(input, weight, act, keep_products and torch.is_grad_enabled())


def linear_cross_entropy(input, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of softmax(input weight^T) against ``target`` without holding the logits;
    ``reduction`` 'mean' (over the rows that are not ignored), 'sum' or 'none'."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none'")
    loss = _LinearCrossEntropy.apply(input, weight, target, ignore_index)
    if reduction == "none":
        return loss
    return loss.sum() / (target != ignore_index).sum() if reduction == "mean" else loss.sum()


def linear_log_probs(input, weight, target, temperature=1.0, ignore_index=-100):
    """(log_prob, entropy) of each row under softmax(input weight^T / temperature), both with
    gradients; 0 where the target is ``ignore_index``."""
    return _LinearLogProbs.apply(input, weight, target, temperature, ignore_index)


__all__ = ["rms_norm", "fused_add_rms_norm", "gated_add_rms_norm", "gated_linear",
           "linear_cross_entropy", "linear_log_probs"]
