"""The differentiable forms against torch's own autograd in 64 bits, and the training example."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

from hp_rms_norm_b200 import autograd as A
from tests import training_reference as R

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_example():
    spec = importlib.util.spec_from_file_location(
        "train_language_model", os.path.join(ROOT, "examples", "train_language_model.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def leaf(*shape, device, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype).requires_grad_()


def doubles(ts):
    return [t.detach().double().requires_grad_() for t in ts]


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("keep", [True, False])
def test_gated_linear(cuda, act, keep):
    x, w = leaf(3, 20, 64, device=cuda, seed=0), leaf(2 * 40, 64, device=cuda, seed=1, scale=0.125)
    y = A.gated_linear(x, w, act, keep_products=keep)
    # sum() hands the backward pass a gradient of one broadcast value.
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    xd, wd = doubles((x, w))
    s = R.gated_linear_backward(torch.ones(60, 40, device=cuda), xd.view(60, 64), wd, act)
    R.assert_near(gx.view(60, 64), s[0].detach(), R.rounding_noise(s[2], wd, x.dtype).detach(), "dx")
    R.assert_near(gw, s[1].detach(), R.rounding_noise(s[2].T, xd.view(60, 64), x.dtype).detach(), "dw")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy(cuda, reduction):
    x, w = leaf(5, 14, 96, device=cuda, seed=2), leaf(333, 96, device=cuda, seed=3, scale=0.2)
    t = torch.randint(0, 333, (5, 14), device=cuda)
    t[0, :3] = -100
    loss = A.linear_cross_entropy(x, w, t, reduction=reduction)
    c = torch.linspace(0.5, 1.5, 70, device=cuda).view(5, 14)
    total = loss if loss.dim() == 0 else (loss * c).sum()
    gx, gw = torch.autograd.grad(total, (x, w))
    xd, wd = doubles((x, w))
    want = torch.nn.functional.cross_entropy((xd @ wd.T).view(70, 333), t.view(70), reduction=reduction)
    # fp32 losses of about 6, from fp32 sums of 96 and 333 terms
    assert (loss.double().view(-1) - want.view(-1)).abs().max() <= 6 * 500 * R.F32
    want = want if want.dim() == 0 else (want * c.view(70).double()).sum()
    wx, ww = torch.autograd.grad(want, (xd, wd))
    counts = (t != -100).view(70)
    rows = c.view(70) if reduction == "none" else torch.ones(70, device=cuda)
    rows = rows / counts.sum() if reduction == "mean" else rows
    s = R.linear_cross_entropy_backward(rows, xd.detach().view(70, 96), wd.detach(), t.view(70), -100)[2]
    R.assert_near(gx, wx, R.rounding_noise(s, wd.detach(), x.dtype).view(5, 14, 96), "dx")
    R.assert_near(gw, ww, R.rounding_noise(s.T, xd.detach().view(70, 96), x.dtype), "dw")


def test_norms(cuda):
    x, r = leaf(7, 9, 320, device=cuda, seed=4), leaf(7, 9, 320, device=cuda, seed=5)
    w = leaf(320, device=cuda, seed=6)
    y, total = A.fused_add_rms_norm(x, r, w, 1e-6)
    y2 = A.rms_norm(total, w, 1e-6)
    before = total.clone()
    gx, gr, gw = torch.autograd.grad((y * y2).sum() + total.sum(), (x, r, w))
    assert torch.equal(gx, gr) and torch.equal(total, before)
    td, wd = doubles((total, w))
    inv = torch.rsqrt(td.square().mean(-1, keepdim=True) + 1e-6)
    n = td * inv * wd
    want_t, want_w = torch.autograd.grad((n * n).sum() + td.sum(), (td, wd))
    # y, y2, each norm's gradient and the sums of two gradients are rounded: four
    # roundings of the terms that the two norms' gradients are made of.
    with torch.no_grad():
        unit, g = (td * inv).abs(), (wd * n).abs()
        size_t = 2 * inv * (g + unit * (g * unit).mean(-1, keepdim=True)) + want_t.abs()
        size_w = 2 * (n * unit).square().sum((0, 1)).sqrt() + want_w.abs()
    R.assert_near(gx, want_t, 4 * R.U[x.dtype] * size_t, "dx")
    R.assert_near(gw, want_w, 4 * R.U[x.dtype] * size_w, "dw")


def test_norm_with_one_of_its_results_used(cuda):
    x, r = leaf(6, 256, device=cuda, seed=7), leaf(6, 256, device=cuda, seed=8)
    w = leaf(256, device=cuda, seed=9)
    c = leaf(6, 256, device=cuda, seed=10).detach()
    y, total = A.fused_add_rms_norm(x, r, w, 1e-6)
    # Only the norm: what a zero gradient for the sum gives.
    got = torch.autograd.grad(y, (x, r, w), c, retain_graph=True)
    want = torch.autograd.grad((y, total), (x, r, w), (c, torch.zeros_like(c)), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Only the sum: its gradient as it is, and none for the weight.
    gx, gr, gw = torch.autograd.grad(total, (x, r, w), c, allow_unused=True)
    assert torch.equal(gx, c) and torch.equal(gr, c) and gw is None


@pytest.mark.parametrize("name", ["rms_norm", "fused_add_rms_norm", "gated_linear", "linear_cross_entropy"])
def test_second_derivatives_are_refused(cuda, name):
    x, w = leaf(4, 64, device=cuda, seed=11), leaf(32, 64, device=cuda, seed=12)
    n = leaf(64, device=cuda, seed=13)
    y = {"rms_norm": lambda: A.rms_norm(x, n, 1e-6),
         "fused_add_rms_norm": lambda: A.fused_add_rms_norm(x, x, n, 1e-6)[0],
         "gated_linear": lambda: A.gated_linear(x, w),
         "linear_cross_entropy": lambda: A.linear_cross_entropy(x, w, torch.tensor([0, 1, 2, 3], device=cuda))}[name]()
    (gx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.float().sum().backward()


def test_example_learns(cuda):
    losses = load_example().train(steps=30, layers=2, hidden=256, ffn=700, vocab=1000, batch=8, length=128)
    losses = losses.cpu()
    # It starts at guessing (the logarithm of the vocabulary) or above.
    assert torch.isfinite(losses).all() and losses[0] > 6.5
    assert losses[-5:].mean() < losses[:5].mean() - 0.5


def test_example_gradients_match_plain_torch(cuda):
    """One backward pass of the example's model against the same model in plain torch, float64."""
    ex = load_example()
    p = ex.parameters(2, 128, 200, 300, cuda, torch.bfloat16)
    tokens = torch.randint(0, 300, (4, 32), device=cuda)
    targets = torch.randint(0, 300, (4, 32), device=cuda)
    loss = ex.loss_of(p, 2, tokens, targets)
    names = list(p)
    grads = torch.autograd.grad(loss, [p[n] for n in names])

    class Plain:
        @staticmethod
        def fused_add_rms_norm(x, r, w, eps):
            t = x + r
            return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w, t

        @staticmethod
        def gated_linear(x, w, act="silu"):
            g, u = (x @ w.T).chunk(2, -1)
            return torch.nn.functional.silu(g) * u

        @staticmethod
        def linear_cross_entropy(x, w, t):
            return torch.nn.functional.cross_entropy((x @ w.T).flatten(0, 1), t.flatten())

    q = {n: p[n].detach().double().requires_grad_() for n in names}
    kept, ex.A = ex.A, Plain
    try:
        want_loss = ex.loss_of(q, 2, tokens, targets)
    finally:
        ex.A = kept
    want = torch.autograd.grad(want_loss, [q[n] for n in names])
    # Some twenty roundings of u = 2^-8 between the embedding and the loss and
    # as many on the way back, independent of each other: sqrt(40) u.
    assert abs(loss.item() - want_loss.item()) <= 40 ** 0.5 * 2 ** -8 * want_loss.item()
    for n, got, exact in zip(names, grads, want):
        rel = float((got.double() - exact).norm() / exact.norm())
        assert rel <= 40 ** 0.5 * 2 ** -8, (n, rel)


def test_first_calls_inside_graph_capture(cuda):
    worker = os.path.join(ROOT, "tests", "graph_first_training_call_worker.py")
    r = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "OK" in r.stdout, r.stderr[-2000:]


def test_offsets_past_32_bits(cuda):
    """A weight of more than 2^31 elements: the last vocabulary rows, and their gradients."""
    import hp_rms_norm_b200 as hp

    rows, hidden, vocab = 5, 2048, 1_050_000
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(rows, hidden, generator=g, device=cuda).bfloat16()
    w = torch.empty(vocab, hidden, dtype=torch.bfloat16, device=cuda)
    w.normal_(0, hidden ** -0.5, generator=g)
    t = torch.tensor([0, 1, vocab - 1, vocab - 2, 777_777], device=cuda)
    loss, lse = hp.linear_cross_entropy(x, w, t)
    logits = torch.cat([x.double() @ p.double().T for p in w.split(70_000)], 1)
    want = torch.logsumexp(logits, 1)
    # fp32 sums of `hidden` terms, and of `vocab` exponentials in float32 tiles
    assert (lse.double() - want).abs().max() <= hidden * R.F32 * 40 + 64 * R.F32 * 20
    assert (loss.double() - (want - logits.gather(1, t[:, None])[:, 0])).abs().max() <= hidden * R.F32 * 80
    c = torch.ones(rows, device=cuda)
    dx, dw = hp.linear_cross_entropy_backward(c, x, w, t, lse)
    s = torch.exp(logits - want[:, None])
    s[torch.arange(rows, device=cuda), t] -= 1
    want_x = sum(a @ p.double() for a, p in zip(s.split(70_000, 1), w.split(70_000)))
    R.assert_near(dx, want_x, R.U[x.dtype] * torch.sqrt(s.square().sum(1, keepdim=True)) * hidden ** -0.5 * 4
                  * torch.ones_like(want_x), "dx")
    for rows_of in (slice(0, 64), slice(777_700, 777_800), slice(vocab - 64, vocab)):
        part = s[:, rows_of].T
        R.assert_near(dw[rows_of], part @ x.double(), R.rounding_noise(part, x.double(), x.dtype), "dw")
    half = vocab // 2
    out = hp.gated_linear(x, w, "silu")
    gate, up = x.double() @ w[half - 50:half].double().T, x.double() @ w[-50:].double().T
    R.assert_near(out[:, -50:], torch.nn.functional.silu(gate) * up, hidden * R.F32 * up.abs(), "gated")
