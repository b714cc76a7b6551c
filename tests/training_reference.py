"""The training operators' formulas in 64 bits, and bounds on how far a kernel may be from them.

A kernel's result differs from the formula by (1) the rounding of 16-bit outputs, at most
u = 2^-8 (bf16) or 2^-11 (fp16) of a value, half an ulp of the smallest normal below it; (2) the
rounding of a 16-bit intermediate S, at most u |S| and so u (|S| |W|) in a sum of products; (3)
fp32 sums of k products, taken in any order: at most k 2^-23 times the sum of magnitudes (twice
the unit roundoff a step, for adders that truncate).  The bounds below add these up; nothing in
them is fitted to what a kernel returns.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
F32 = 2.0 ** -23


def act_and_slope(a, act):
    if act == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    if act == "gelu":
        p = 0.5 * torch.erfc(-a / math.sqrt(2))
        return a * p, p + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    k, c = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(k * (a + c * a ** 3))
    return a * (1 + t) / 2, (1 + t) / 2 + a * (1 - t * t) * k * (1 + 3 * c * a * a) / 2


def gated_linear(x, w, act):
    """(out, gate, up)"""
    x, w = x.double(), w.double()
    d = w.shape[0] // 2
    gate, up = x @ w[:d].T, x @ w[d:].T
    return act_and_slope(gate, act)[0] * up, gate, up


def gated_linear_backward(dout, x, w, act):
    """(dx, dw, S)"""
    _, gate, up = gated_linear(x, w, act)
    value, slope = act_and_slope(gate, act)
    dout = dout.double()
    s = torch.cat((dout * up * slope, dout * value), -1)
    return s @ w.double(), s.T @ x.double(), s


def linear_cross_entropy(x, w, target, ignore):
    """(loss, lse, logits)"""
    logits = x.double() @ w.double().T
    lse = torch.logsumexp(logits, -1)
    counts = target != ignore
    at = torch.where(counts, target, 0)
    loss = torch.where(counts, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    return loss, lse, logits


def linear_cross_entropy_backward(c, x, w, target, ignore):
    """(dx, dw, S)"""
    _, lse, logits = linear_cross_entropy(x, w, target, ignore)
    counts = target != ignore
    s = torch.exp(logits - lse[:, None])
    s[torch.arange(len(target), device=s.device), torch.where(counts, target, 0)] -= 1
    s = s * (c.double() * counts)[:, None]
    return s @ w.double(), s.T @ x.double(), s


def rms_norm_backward(dy, x, w, eps, extra=None):
    """(dx, dw)"""
    dy, x, w = dy.double(), x.double(), w.double()
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n, g = x * inv, dy * w
    dx = inv * (g - n * (g * n).mean(-1, keepdim=True))
    return dx if extra is None else dx + extra.double(), (dy * n).sum(0)


def clip(grads, max_norm):
    """(norm, clipped)"""
    norm = torch.sqrt(sum(g.double().square().sum() for g in grads))
    return norm, [g.double() * min(1.0, max_norm / (norm.item() + 1e-6)) for g in grads]


# ---------------------------------------------------------------------------

def assert_within(got, want, bound, label):
    err = (got.double() - want).abs()
    over = err > bound
    assert not over.any(), (
        f"{label}: {int(over.sum())} of {over.numel()} values out of bounds, worst "
        f"{float((err / bound.clamp(min=1e-300)).max()):.3g} of the bound")


def assert_near(got, want, noise, label):
    """The error's norm: the output's own rounding, at most u a value, and `noise`, the size
    that the errors before it have in each value (0 for none)."""
    allowed = 1.01 * U[got.dtype] * float(want.norm()) + float(torch.as_tensor(noise).norm())
    err = float((got.double() - want).norm())
    assert err <= allowed, f"{label}: error of norm {err:.3g}, at most {allowed:.3g}"


def rounding_noise(s, w, dtype):
    """The size of sum_k dS_k W_k for roundings |dS_k| <= u |S_k| that are independent of each
    other: u times the root of the sum of squares.  (Relative to the terms: where these cancel
    it is not small against the sum.)"""
    return U[dtype] * torch.sqrt(s.square() @ w.square())


def product_bound(s, w, s_error, depth):
    """How far fp32 sums of (S + dS) W may be from S W, |dS| <= s_error."""
    return s_error @ w.abs() + depth * F32 * ((s.abs() + s_error) @ w.abs())


def rounded(bound, want, dtype):
    return bound + U[dtype] * (want.abs() + bound) + TINY[dtype]
