"""The operators around a block run together: a block in 8-bit integers scored for its tokens, and a
training step of gated blocks under a policy-gradient loss; their waits made to run out; their first
calls inside a capture."""
import os
import subprocess
import sys

import pytest
import torch

import hp_rms_norm_b200 as hp
from hp_rms_norm_b200 import autograd as A
from hp_rms_norm_b200 import capi
from tests import block_reference as B
from tests import training_reference as R

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6


def quantised(w):
    scale = w.abs().amax(1) / 127
    return torch.round(w / scale[:, None]).to(torch.int8), scale


def product(codes, scale, weight, weight_scale):
    """The integers' sums first, which 64 bits hold exactly: scales multiplied into the terms would
    leave 2^-53 of the terms' size where the sum is 0."""
    return (codes.double() @ weight.double().T) * scale.double()[:, None] * weight_scale.double()


@pytest.mark.parametrize("tokens", [1, 5, 64, 300])
def test_scoring_a_quantised_block(cuda, tokens):
    """norm -> int8 products -> gated activation -> int8 product -> gated norm -> log probabilities,
    each stage's output against the 64-bit formula of that stage's inputs."""
    g = torch.Generator(device=cuda).manual_seed(tokens)
    hidden, ffn, vocab = 512, 704, 5000
    normal = lambda *s, scale=1.0: torch.randn(*s, generator=g, device=cuda) * scale  # noqa: E731
    x, residual = normal(tokens, hidden).bfloat16(), normal(tokens, hidden, scale=2.0).bfloat16()
    norms = [(1 + normal(hidden, scale=0.1)).bfloat16() for _ in range(3)]
    gate = normal(hidden, scale=0.5).bfloat16()
    up, up_scale = quantised(normal(2 * ffn, hidden, scale=hidden ** -0.5))
    down, down_scale = quantised(normal(hidden, ffn, scale=ffn ** -0.5))
    head = normal(vocab, hidden, scale=2 * hidden ** -0.5).bfloat16()
    target = torch.randint(0, vocab, (tokens,), generator=g, device=cuda)

    total = torch.empty_like(residual)
    q, s = hp.rms_norm_int8(x, norms[0], EPS, residual=residual, residual_out=total)
    gate_up = hp.linear_int8(q, s, up, up_scale)
    want = product(q, s, up, up_scale)
    R.assert_within(gate_up, want, R.rounded(3 * R.F32 * want.abs(), want, gate_up.dtype), "gate and up")
    h, hs = hp.quantize_int8(hp.silu_and_mul(gate_up))
    y = hp.linear_int8(h, hs, down, down_scale)
    want = product(h, hs, down, down_scale)
    R.assert_within(y, want, R.rounded(3 * R.F32 * want.abs(), want, y.dtype), "down")
    (out_want, bound), (total_want, total_bound) = B.gated_add_rms_norm(y, total, norms[1], norms[2], EPS, gate)
    out = hp.gated_add_rms_norm(y, total, norms[1], norms[2], EPS, gate=gate)
    R.assert_within(total, total_want, R.rounded(total_bound, total_want, total.dtype), "residual")
    R.assert_within(out, out_want, R.rounded(bound, out_want, out.dtype), "out")
    found = hp.linear_log_probs(out, head, target, top=3)
    log_prob, entropy, _, logits = B.log_probs(out, head, target, -100)
    each, lse_err, entropy_err = B.log_prob_errors(out, head)
    R.assert_within(found.log_prob, log_prob, lse_err + each.max(-1).values + 4 * R.F32 * 20, "log_prob")
    R.assert_within(found.entropy, entropy, entropy_err, "entropy")
    assert torch.equal(found.top_indices, logits.sort(dim=-1, descending=True, stable=True).indices[:, :3])


def test_training_step_of_gated_blocks(cuda):
    """Gradients of a stack of gated blocks and a policy-gradient loss with an entropy term against
    the same step in 64 bits by automatic differentiation."""
    g = torch.Generator(device=cuda).manual_seed(0)
    batch, length, hidden, ffn, vocab, layers = 3, 40, 128, 192, 700, 2
    dt = torch.float16
    normal = lambda *s, scale=1.0, mean=0.0: (torch.randn(*s, generator=g, device=cuda) * scale + mean).to(dt)  # noqa: E731
    p = {"x": normal(batch, length, hidden), "head": normal(vocab, hidden, scale=2 * hidden ** -0.5)}
    for k in range(layers):
        p |= {f"up{k}": normal(2 * ffn, hidden, scale=hidden ** -0.5), f"down{k}": normal(hidden, ffn, scale=ffn ** -0.5),
              f"post{k}": normal(hidden, scale=0.1, mean=0.7), f"pre{k}": normal(hidden, scale=0.1, mean=1.0),
              f"gate{k}": normal(batch, 1, hidden, scale=0.2, mean=0.8)}
    p = {k: v.requires_grad_() for k, v in p.items()}
    target = torch.randint(0, vocab, (batch, length), generator=g, device=cuda)
    target[torch.rand(batch, length, generator=g, device=cuda) < 0.3] = -100
    advantage = torch.randn(batch, length, generator=g, device=cuda)

    def ours(p):
        total = p["x"]
        y = A.rms_norm(total, p["pre0"], EPS)
        for k in range(layers):
            z = torch.nn.functional.linear(A.gated_linear(y, p[f"up{k}"]), p[f"down{k}"])
            y, total = A.gated_add_rms_norm(z, total, p[f"post{k}"], p[f"pre{k}"], EPS, gate=p[f"gate{k}"], residual_scale=0.9)
        log_prob, entropy = A.linear_log_probs(y, p["head"], target, temperature=0.8)
        return -(advantage * log_prob + 0.01 * entropy).sum()

    def exact(p):
        norm = lambda a, w: a * torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS) * w  # noqa: E731
        total = p["x"]
        y = norm(total, p["pre0"])
        for k in range(layers):
            a, b = (y @ p[f"up{k}"].T).chunk(2, -1)
            z = (torch.nn.functional.silu(a) * b) @ p[f"down{k}"].T
            total = 0.9 * total + p[f"gate{k}"] * norm(z, p[f"post{k}"])
            y = norm(total, p[f"pre{k}"])
        log_p = torch.log_softmax(y @ p["head"].T / 0.8, -1)
        counts = target != -100
        log_prob = log_p.gather(-1, target.clamp(min=0)[..., None])[..., 0] * counts
        return -(advantage.double() * log_prob + 0.01 * -(log_p.exp() * log_p).sum(-1) * counts).sum()

    got = torch.autograd.grad(ours(p), list(p.values()))
    wide = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    want = torch.autograd.grad(exact(wide), list(wide.values()))
    # Some 12 roundings to 16 bits lie between a leaf and its gradient (activations, residuals and
    # gradients of each layer), each at most u of what it rounds and independent of the others; the
    # layers' factors (norms of random weights, about 1; gates and residuals below 2) leave their size.
    for name, a, b in zip(p, got, want):
        assert (a.double() - b).norm() <= 12 * 2 * R.U[dt] * b.norm(), name
    # And into the optimiser's buffers.
    out = [torch.empty_like(v, dtype=torch.float32) for v in got]
    norm = hp.clip_grad_norm(list(got), 1.0, out=out)
    assert torch.isfinite(norm) and torch.stack([v.norm() for v in out]).norm() <= 1.0 + 1e-5


def block(rows, hidden, start, gate, device):
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(start + rows * hidden, generator=g, device=device).bfloat16()[start:].view(rows, hidden)
    w = x[0].clone()
    gates = {"none": None, "channel": w, "sequence": x.view(-1, 10, hidden)[:, :1].contiguous(), "full": x.clone()}[gate]
    y = x.view(-1, 10, hidden) if gate == "sequence" else x
    return lambda: [v for v in hp.gated_add_rms_norm_backward(y, y, y, w, w, EPS, gate=gates, grad_residual=y) if v is not None]


def probs(rows, hidden, vocab, top, device):
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(rows, hidden, generator=g, device=device).half()
    w = (torch.randn(vocab, hidden, generator=g, device=device) / 16).half()
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    return lambda: [v for v in hp.linear_log_probs(x, w, t, top=top) if v is not None]


def int8(rows, hidden, channels, device):
    g = torch.Generator(device=device).manual_seed(rows)
    x, w = (torch.randint(-127, 128, (n, hidden), generator=g, device=device, dtype=torch.int8) for n in (rows, channels))
    xs, ws = torch.rand(rows, generator=g, device=device), torch.rand(channels, generator=g, device=device)
    return lambda: (hp.linear_int8(x, xs, w, ws),)


CALLS = {"norm": (block, 700, 1024, 0, "channel"), "norm long": (block, 300, 16384, 0, "none"), "norm wide": (block, 300, 8192, 0, "full"),
         "norm odd": (block, 700, 1001, 1, "channel"), "norm sequences": (block, 700, 512, 0, "sequence"),
         "log probabilities": (probs, 2048, 640, 6000, 0), "log probabilities few": (probs, 40, 100, 3000, 0),
         "8-bit": (int8, 700, 512, 640), "8-bit shares": (int8, 40, 8192, 300)}


@pytest.mark.parametrize("name", list(CALLS))
def test_waits_that_run_out(cuda, name):
    """The hook leaves out all loads, so every role gives up after 5 ms: the launch ends, the count
    tells, later calls are refused until it is reset, and nothing is left behind."""
    make, *sizes = CALLS[name]
    call = make(*sizes, cuda)
    want = call()
    torch.cuda.synchronize()
    assert capi.wait_timeouts(reset=True) == 0
    try:
        capi.test_stall_loads(True, 5_000_000)
        call()
        torch.cuda.synchronize()
    finally:
        capi.test_stall_loads(False)
    assert capi.wait_timeouts() > 0
    for _ in range(2):
        with pytest.raises(RuntimeError, match="ran out"):
            call()
    assert capi.wait_timeouts(reset=True) > 0
    got = call()
    torch.cuda.synchronize()
    assert capi.wait_timeouts() == 0
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_first_calls_inside_a_capture(cuda):
    worker = os.path.join(ROOT, "tests", "graph_first_block_call_worker.py")
    r = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("OK"), r.stdout + r.stderr


def test_calls_at_once_on_two_streams(cuda):
    """The same tensors through both streams, workspaces of their own."""
    calls = [make(*sizes, cuda) for make, *sizes in (CALLS["norm"], CALLS["log probabilities"], CALLS["8-bit shares"])]
    calls.append(probs(64, 128, 5000, 8, cuda))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append([c() for c in calls])
    torch.cuda.synchronize()
    for side in got:
        for found in side:
            for a, b in zip(want, found):
                assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_outputs_have_no_history(cuda):
    """Weights that ask for gradients, in calls outside the differentiable forms."""
    x = torch.randn(4, 64, device=cuda).bfloat16()
    w = torch.randn(50, 64, device=cuda).bfloat16().requires_grad_()
    t = torch.zeros(4, dtype=torch.int64, device=cuda)
    found = hp.linear_log_probs(x, w, t, top=2)
    assert not any(v.requires_grad for v in found)
    assert not any(v.requires_grad for v in hp.rms_norm_int8(x, w[0], EPS))


def test_compiled(cuda):
    """Traced without a break, the same results."""
    x, r = torch.randn(8, 256, device=cuda).bfloat16(), torch.randn(8, 256, device=cuda).bfloat16()
    w = torch.ones(256, device=cuda).bfloat16()
    w8, ws = torch.randint(-127, 128, (64, 256), device=cuda, dtype=torch.int8), torch.rand(64, device=cuda)

    def f(x, r):
        total = torch.empty_like(r)
        out = hp.gated_add_rms_norm(x, r, w, w, EPS, gate=w, residual_out=total)
        q, s = hp.rms_norm_int8(out, w, EPS)
        return out, total, hp.linear_int8(q, s, w8, ws)

    want = f(x, r)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x, r)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
