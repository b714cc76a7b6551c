"""rms_norm_backward on the GPU against the 64-bit formula."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from tests import training_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 256), (37, 1000), (64, 5001), (130, 128), (300, 2056),
          (1000, 64), (257, 8192), (9, 16384), (20, 32768), (3, 40001), (2, 70000)]


def make(rows, hidden, dtype, device, pad=0):
    g = torch.Generator(device=device).manual_seed(rows * 7 + hidden)
    wide = lambda: torch.randn(rows, hidden + pad, generator=g, device=device).to(dtype)[:, :hidden]
    x, dy, extra = wide(), wide(), wide()
    w = (1 + 0.1 * torch.randn(hidden, generator=g, device=device)).to(dtype)
    return x, dy, extra, w


def check(dx, dw, dy, x, w, eps, extra, label):
    want_x, want_w = R.rms_norm_backward(dy, x, w, eps, extra)
    rows, hidden = x.shape
    xd, g = x.double(), (dy.double() * w.double()).abs()
    inv = torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps)
    n = (xd * inv).abs()
    k = (hidden + 16) * R.F32  # fp32 sums of `hidden` terms, and a dozen more operations
    bound = k * inv * (g + n * (g * n).mean(-1, keepdim=True)) * 2
    if extra is not None:
        bound = bound + 2 * R.F32 * (extra.double().abs() + want_x.abs())
    R.assert_within(dx, want_x, R.rounded(bound, want_x, dx.dtype), label + " dx")
    R.assert_near(dx, want_x, bound, label + " dx")
    bound = (rows + 2 * hidden + 16) * R.F32 * (dy.double().abs() * n).sum(0)
    R.assert_within(dw, want_w, R.rounded(bound, want_w, dw.dtype), label + " dw")
    R.assert_near(dw, want_w, bound, label + " dw")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(cuda, shape, dt):
    x, dy, extra, w = make(*shape, DTYPES[dt], cuda)
    for e in (None, extra):
        dx, dw = hp.rms_norm_backward(dy, x, w, 1e-6, grad_residual=e)
        check(dx, dw, dy, x, w, 1e-6, e, f"{shape} {dt} {e is not None}")


@pytest.mark.parametrize("pad", [1, 2, 8])
def test_strided_rows(cuda, pad):
    x, dy, extra, w = make(50, 1000, torch.bfloat16, cuda, pad=pad)
    dx, dw = hp.rms_norm_backward(dy, x, w, 1e-5, grad_residual=extra)
    check(dx, dw, dy, x, w, 1e-5, extra, f"pad {pad}")


def test_zero_rows_and_outliers(cuda):
    x, dy, extra, w = make(40, 640, torch.bfloat16, cuda)
    x[3] = 0  # inv = 1 / sqrt(eps)
    x[4, 5] = 5000.0
    dx, dw = hp.rms_norm_backward(dy, x, w, 1e-6)
    check(dx, dw, dy, x, w, 1e-6, None, "zero row")
    x[7, 0] = float("nan")
    got, _ = hp.rms_norm_backward(dy, x, w, 1e-6)
    keep = torch.arange(40, device=cuda) != 7
    assert torch.equal(got[keep], dx[keep]) and got[7].isnan().all()


def test_fused_form_matches_autograd(cuda):
    """The gradient through residual += input; y = RMSNorm(residual) w, residual used again."""
    x, dy, extra, w = make(24, 512, torch.bfloat16, cuda)
    res = extra.clone()
    hp.fused_add_rms_norm(x, res, w, 1e-6)
    dx, dw = hp.rms_norm_backward(dy, res, w, 1e-6, grad_residual=extra)
    r, wd = res.double().requires_grad_(), w.double().requires_grad_()
    y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-6) * wd
    gr, gw = torch.autograd.grad((y * dy.double()).sum() + (r * extra.double()).sum(), (r, wd))
    R.assert_near(dx, gr, 0.0, "dx")
    R.assert_near(dw, gw, 0.0, "dw")


def test_repeats_streams_graphs_empty(cuda):
    x, dy, extra, w = make(600, 1024, torch.float16, cuda)
    want = hp.rms_norm_backward(dy, x, w, 1e-6, extra)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = hp.rms_norm_backward(dy, x, w, 1e-6, extra)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = hp.rms_norm_backward(dy, x, w, 1e-6, extra)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, kept):
        assert torch.equal(a, b) and torch.equal(a, c)
    dx, dw = hp.rms_norm_backward(dy[:0], x[:0], w, 1e-6)
    assert dx.shape == (0, 1024) and not dw.any()


def test_refusals(cuda):
    x, dy, extra, w = make(4, 32, torch.bfloat16, cuda)
    for bad in (lambda: hp.rms_norm_backward(dy[:3], x, w, 1e-6),
                lambda: hp.rms_norm_backward(dy.half(), x, w, 1e-6),
                lambda: hp.rms_norm_backward(dy, x, w[:5], 1e-6),
                lambda: hp.rms_norm_backward(dy.float(), x.float(), w.float(), 1e-6),
                lambda: hp.rms_norm_backward(dy, x, w, 1e-6, grad_residual=extra[:, :5]),
                lambda: hp.rms_norm_backward(dy.cpu(), x, w, 1e-6)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("hidden", [501, 5001])
@pytest.mark.parametrize("start", [1, 6])
def test_ends_off_boundaries_and_buffers_used_again(cuda, hidden, start):
    """Tensors whose first and last elements lie inside a 16-byte granule, with enough rows that
    the buffers which took these elements one by one are filled by copies later."""
    rows = 6000
    g = torch.Generator(device=cuda).manual_seed(hidden + start)
    odd = lambda: torch.randn(start + rows * hidden, generator=g, device=cuda).bfloat16()[start:].view(rows, hidden)
    x, dy, extra = odd(), odd(), odd()
    w = (1 + 0.1 * torch.randn(hidden, generator=g, device=cuda)).bfloat16()
    for e in (None, extra):
        dx, dw = hp.rms_norm_backward(dy, x, w, 1e-6, grad_residual=e)
        check(dx, dw, dy, x, w, 1e-6, e, f"{hidden} {start} {e is not None}")
        again = hp.rms_norm_backward(dy, x, w, 1e-6, grad_residual=e)
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
