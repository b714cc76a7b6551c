"""64-bit formulas of the operators around a block (the gated norms, log probabilities of tokens,
8-bit integer products), with bounds on how far fp32 kernels may be from them.

As in training_reference.py a bound adds up (1) the rounding of 16-bit outputs, (2) that of 16-bit
intermediates, (3) fp32 operations, 2^-23 of the value each (twice the unit roundoff) and, for
sums, times the additions on the longest path: a thread adds up at most hidden / 256 + 32 terms
before at most 32 sums join, so `path` below.
"""
from __future__ import annotations

import torch

from tests.training_reference import F32, U, rounded  # noqa: F401


def path(n):
    return n / 256 + 64


def spread_gate(gate, x):
    """The gate over x's shape, in 64 bits; 1 without one."""
    return torch.ones_like(x) if gate is None else gate.double().expand(x.shape)


def inv_rms(x, eps):
    return torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def gated_add_rms_norm(x, r, p, w, eps, gate=None, scale=1.0):
    """((out, bound), (total, bound)), the bounds without the outputs' rounding."""
    x, r, w = x.double(), r.double(), w.double()
    rel = (path(x.shape[-1]) / 2 + 4) * F32  # of an inverse root of a mean of squares
    y = spread_gate(gate, x) * (x if p is None else x * inv_rms(x, eps) * p.double())
    total = scale * r + y
    total_bound = y.abs() * (rel + 4 * F32) + F32 * ((scale * r).abs() + total.abs())
    inv = inv_rms(total, eps)
    out = total * inv * w
    # 1 / inv is at least the root mean square of total: how far errors in it move inv.
    moved = total_bound.square().mean(-1, keepdim=True).sqrt() * inv
    out_bound = total_bound * inv * w.abs() + out.abs() * (moved + rel + 3 * F32)
    return (out, out_bound), (total, total_bound)


def gated_add_rms_norm_backward(d, x, t, p, w, eps, gate=None, scale=1.0, e=None):
    """{name: (gradient, bound)} for the new residual t as it was written."""
    d, x, t, w = d.double(), x.double(), t.double(), w.double()
    e = torch.zeros_like(t) if e is None else e.double()
    h, rows = x.shape[-1], max(1, x.numel() // max(1, x.shape[-1]))
    rel = (path(h) / 2 + 4) * F32
    g = spread_gate(gate, x)
    pp = torch.ones_like(x) if p is None else p.double().expand(x.shape)
    inv_t = inv_rms(t, eps)
    inv_x = torch.ones_like(inv_t) if p is None else inv_rms(x, eps)
    n, m = t * inv_t, x * inv_x
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    c1 = mean(w * d * n)
    c1_err = mean((w * d * n).abs()) * (path(h) * F32 + rel + 4 * F32)
    dt = inv_t * (w * d - n * c1) + e
    dt_err = inv_t * (n.abs() * c1_err + ((n * c1).abs() + (w * d).abs()) * (2 * rel + 4 * F32)) + 2 * F32 * (dt.abs() + e.abs())
    u = pp * g * dt
    u_err = (pp * g).abs() * dt_err + 2 * F32 * u.abs()
    if p is None:
        dx, dx_err = u, u_err
    else:
        c2 = mean(u * m)
        c2_err = mean(m.abs() * u_err) + mean((u * m).abs()) * (path(h) * F32 + rel + 4 * F32)
        dx = inv_x * (u - m * c2)
        dx_err = inv_x * (u_err + m.abs() * c2_err + ((m * c2).abs() + u.abs()) * (2 * rel + 4 * F32))
    lead = tuple(range(x.dim() - 1))
    found = {"x": (dx, dx_err), "residual": (scale * dt, abs(scale) * dt_err + F32 * (scale * dt).abs())}
    found["weight"] = ((d * n).sum(lead), (d * n).abs().sum(lead) * (rel + (rows + 2) * F32))
    if p is not None:
        s = g * dt * m
        s_err = (g * m).abs() * dt_err + s.abs() * (rel + 3 * F32)
        found["post_weight"] = (s.sum(lead), s_err.sum(lead) + (rows + 2) * F32 * s.abs().sum(lead))
    if gate is not None:
        s = dt * m * pp
        s_err = (m * pp).abs() * dt_err + s.abs() * (rel + 3 * F32)
        shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
        over = [k for k in range(x.dim()) if shape[k] == 1 and x.shape[k] != 1]
        count = max(1, x.numel() // max(1, gate.numel()))
        reduce = lambda v: (v.sum(over, keepdim=True) if over else v).reshape(gate.shape)  # noqa: E731
        found["gate"] = (reduce(s), reduce(s_err) + (count + 2) * F32 * reduce(s.abs()))
    return found


def log_probs(x, w, target, ignore, temperature=1.0):
    """(log_prob, entropy, lse, logits)"""
    logits = x.double() @ w.double().T / temperature
    lse = torch.logsumexp(logits, -1)
    log_p = logits - lse[:, None]
    counts = target != ignore
    at = torch.where(counts, target, 0)
    log_prob = torch.where(counts, log_p.gather(1, at[:, None])[:, 0], 0.0)
    entropy = torch.where(counts, -(log_p.exp() * log_p).sum(-1), 0.0)
    return log_prob, entropy, lse, logits


def log_prob_errors(x, w, temperature=1.0):
    """(logits' error, lse's, entropy's) of fp32 sums: products of k terms by k 2^-23 of the sum of
    magnitudes; exponentials 2^-21 (2 + the exponent) of themselves; sums over the vocabulary."""
    logits = x.double() @ w.double().T / temperature
    each = (x.shape[1] + 2) * F32 * (x.double().abs() @ w.double().abs().T) / temperature
    vocab = w.shape[0]
    lse = torch.logsumexp(logits, -1)
    e = each.max(-1).values
    spread = (logits.max(-1).values - logits.min(-1).values).clamp(min=1)
    sums = vocab * F32 + 4 * F32 * (2 + spread)
    lse_err = e + sums + 2 * F32 * lse.abs()
    log_p = logits - lse[:, None]
    entropy = -(log_p.exp() * log_p).sum(-1)
    below = logits.max(-1).values - (log_p.exp() * logits).sum(-1)  # the mean distance from the largest
    # The entropy moves by p |log p + entropy| with each logit, 2 entropy in all; it is log s - a / s
    # of sums that are off by `sums`, terms of a by as much again.
    entropy_err = 2 * (entropy + 1) * e + sums * (1 + 3 * below) + 4 * F32 * (1 + below + entropy)
    return each, lse_err, entropy_err


def log_probs_backward(g, x, w, target, ignore, temperature=1.0, h=None):
    """(dx, dw, S, S's error before it is rounded to 16 bits)"""
    _, entropy, lse, logits = log_probs(x, w, target, ignore, temperature)
    each, lse_err, entropy_err = log_prob_errors(x, w, temperature)
    counts = (target != ignore)[:, None]
    log_p = logits - lse[:, None]
    p = log_p.exp()
    off = each + lse_err[:, None] + 4 * F32 * (2 + log_p.abs())
    at = torch.zeros_like(p)
    at[torch.arange(len(target), device=p.device), torch.where(target != ignore, target, 0)] = 1
    g = g.double()[:, None]
    s = g * (at - p)
    err = g.abs() * (p * 2 * off + F32)
    if h is not None:
        h = h.double()[:, None]
        by = log_p + entropy[:, None]
        s = s - h * p * by
        err = err + h.abs() * p * (by.abs() * 2 * off + off + entropy_err[:, None] + 3 * F32 * (log_p.abs() + by.abs()))
    s, err = s * counts / temperature, err * counts / temperature + 2 * F32 * (s * counts).abs() / temperature
    return s @ w.double(), s.T @ x.double(), s, err


def rms_norm_int8(x, w, eps, r=None):
    """(y, how far fp32 operations may be from it, total)"""
    total = x.double() if r is None else x.double() + r.double()
    if w is None:
        return total, F32 * total.abs(), total
    y = total * inv_rms(total, eps) * w.double()
    return y, y.abs() * ((path(x.shape[-1]) / 2 + 4) * F32 + 4 * F32), total
