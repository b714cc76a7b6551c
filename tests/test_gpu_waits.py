"""The training operators' bounded waits, made to run out on purpose: the test hook leaves out all
loads, so every role of a CTA gives up after 5 ms.  The launch ends, the count tells, and later calls
are refused until it is reset; nothing is left behind that a call after that would notice."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from hp_rms_norm_b200 import capi

pytestmark = pytest.mark.gpu


def gated(rows, hidden, d, device):
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(rows, hidden, generator=g, device=device).bfloat16()
    w = (torch.randn(2 * d, hidden, generator=g, device=device) / 16).bfloat16()
    return lambda: (hp.gated_linear(x, w),)


def loss(rows, hidden, vocab, device):
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(rows, hidden, generator=g, device=device).half()
    w = (torch.randn(vocab, hidden, generator=g, device=device) / 16).half()
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    return lambda: hp.linear_cross_entropy(x, w, t)


def norm(rows, hidden, start, device):
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(start + rows * hidden, generator=g, device=device).bfloat16()[start:].view(rows, hidden)
    return lambda: hp.rms_norm_backward(x, x, x[0].clone(), 1e-6, grad_residual=x)


# Single CTAs and pairs, sums in segments, rows with and without 16-byte boundaries, one and
# several rows at once.
CALLS = {"gated token": (gated, 1, 512, 640), "gated batch": (gated, 4096, 256, 2048),
         "loss few": (loss, 7, 1024, 3000), "loss many": (loss, 2048, 640, 6000),
         "norm": (norm, 700, 1024, 0), "norm long": (norm, 300, 16384, 0), "norm odd": (norm, 700, 1001, 1),
         "norm one row each": (norm, 40, 512, 0)}


@pytest.mark.parametrize("name", list(CALLS))
def test_waits_that_run_out(cuda, name):
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
