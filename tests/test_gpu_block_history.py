"""The operators around a block and autograd's bookkeeping: a call outside the differentiable forms says
that its outputs have no history; what traced calls write."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from hp_rms_norm_b200 import autograd as A

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture()
def said(capfd):
    """The notes of a call (what operators write from C++ goes to stderr), each of them every time."""
    before = torch.is_warn_always_enabled()
    torch.set_warn_always(True)

    def of(call):
        capfd.readouterr()
        call()
        return [line for line in capfd.readouterr().err.splitlines() if "have no history" in line]

    yield of
    torch.set_warn_always(before)


def calls(device):
    x, r = torch.randn(4, 64, device=device).bfloat16(), torch.randn(4, 64, device=device).bfloat16()
    w, v = torch.ones(64, device=device).bfloat16(), torch.randn(50, 64, device=device).bfloat16()
    w8, ws = torch.ones(8, 64, dtype=torch.int8, device=device), torch.ones(8, device=device)
    x8, xs, b = torch.ones(4, 64, dtype=torch.int8, device=device), torch.ones(4, device=device), torch.zeros(8, device=device).bfloat16()
    t = torch.zeros(4, dtype=torch.int64, device=device)
    lse, g = torch.ones(4, device=device), torch.ones(4, device=device)
    return {"gated_add_rms_norm_backward": ((x, w), lambda: hp.gated_add_rms_norm_backward(x, x, r, w, w, EPS)),
            "linear_log_probs": ((x, v), lambda: hp.linear_log_probs(x, v, t)),
            "linear_log_probs_backward": ((g, v), lambda: hp.linear_log_probs_backward(g, x, v, t, lse)),
            "rms_norm_int8": ((w, r), lambda: hp.rms_norm_int8(x, w, EPS, residual=r)),
            "rms_norm_int8 into another": ((x, r), lambda: hp.rms_norm_int8(x, w, EPS, residual=r, residual_out=torch.empty_like(r))),
            "linear_int8": ((ws, b), lambda: hp.linear_int8(x8, xs, w8, ws, bias=b))}


@pytest.mark.parametrize("name", list(calls("cpu")))
def test_calls_without_history_say_so(cuda, said, name):
    inputs, call = calls(cuda)[name]
    assert said(call) == []
    for t in inputs:
        t.requires_grad_()
        (text,) = said(call)
        assert "hp_rms_norm::" + name.split()[0] in text
        with torch.no_grad():
            assert said(call) == []
        t.requires_grad_(False)


def test_the_differentiable_forms_say_nothing(cuda, said):
    x, w = torch.randn(4, 64, device=cuda).bfloat16().requires_grad_(), torch.ones(64, device=cuda).bfloat16().requires_grad_()
    v, t = torch.randn(50, 64, device=cuda).bfloat16().requires_grad_(), torch.zeros(4, dtype=torch.int64, device=cuda)

    def step():
        out, total = A.gated_add_rms_norm(x, x, w, w, EPS, gate=w)
        log_prob, entropy = A.linear_log_probs(out, v, t)
        ((log_prob + entropy).sum() + total.float().sum()).backward()

    assert said(step) == []
    assert x.grad is not None and w.grad is not None and v.grad is not None


def test_traced_calls_with_a_residual_of_their_own(cuda):
    """The residual is read after the calls that leave it as it is, and after one that updates it."""
    x, r = torch.randn(4, 256, device=cuda).bfloat16(), torch.randn(4, 256, device=cuda).bfloat16()
    w = torch.ones(256, device=cuda).bfloat16()

    def f(x, r):
        total, other = torch.empty_like(r), torch.empty_like(r)
        out = hp.gated_add_rms_norm(x, r, w, w, EPS, residual_out=total)
        codes, scales = hp.rms_norm_int8(out, w, EPS, residual=r, residual_out=other)
        twice = r * 2
        hp.gated_add_rms_norm(x, twice, w, w, EPS, residual_out=twice)
        hp.rms_norm_int8(x, w, EPS, residual=r)
        return out, total, codes, scales, other, twice, r

    want = f(x, r.clone())
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x, r.clone())
    assert all(torch.equal(a, b) for a, b in zip(want, got))
