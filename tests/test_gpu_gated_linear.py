"""gated_linear and its backward pass on the GPU against the 64-bit formulas."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from tests import training_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# rows x hidden x d: single tokens, ragged rows, sums of odd and of aligned length, a width of one
SHAPES = [(1, 64, 32), (1, 1001, 77), (2, 8, 1), (3, 1, 5), (5, 256, 300), (8, 520, 129),
          (17, 40, 200), (64, 512, 512), (100, 1000, 333), (128, 64, 128), (129, 136, 257),
          (300, 2056, 192), (513, 264, 1000)]


def make(rows, hidden, d, dtype, device, pad=0, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + rows * 7 + hidden * 3 + d)
    x = torch.randn(rows, hidden + pad, generator=g, device=device).to(dtype)[:, :hidden]
    w = (torch.randn(2 * d, hidden, generator=g, device=device) * hidden ** -0.5).to(dtype)
    dout = torch.randn(rows, d, generator=g, device=device).to(dtype)
    return x, w, dout


def check_forward(out, x, w, act, label):
    want, gate, up = R.gated_linear(x, w, act)
    k = x.shape[1]
    xa, wa, d = x.double().abs(), w.double().abs(), w.shape[0] // 2
    eg, eu = k * R.F32 * (xa @ wa[:d].T), k * R.F32 * (xa @ wa[d:].T)
    value = R.act_and_slope(gate, act)[0].abs()
    # |act'| <= 1.13; the activation's own fp32 arithmetic: 8 ulp of |gate| at most.
    ev = 1.13 * eg + 8 * R.F32 * gate.abs()
    bound = ev * (up.abs() + eu) + value * eu
    R.assert_within(out, want, R.rounded(bound, want, out.dtype), label)
    R.assert_near(out, want, bound, label)


def check_backward(dx, dw, dout, x, w, act, label):
    want_x, want_w, s = R.gated_linear_backward(dout, x, w, act)
    _, gate, up = R.gated_linear(x, w, act)
    k, d = x.shape[1], w.shape[0] // 2
    xa, wa, da = x.double().abs(), w.double().abs(), dout.double().abs()
    eg, eu = k * R.F32 * (xa @ wa[:d].T), k * R.F32 * (xa @ wa[d:].T)
    value, slope = R.act_and_slope(gate, act)
    # |act''| <= 1.2; slopes are sums of terms up to 1.2 (1 + |gate|), 8 ulp of these.
    es = 1.2 * eg + 8 * R.F32 * 1.2 * (1 + gate.abs())
    ev = 1.13 * eg + 8 * R.F32 * gate.abs()
    e = torch.cat((da * (es * (up.abs() + eu) + slope.abs() * eu), da * ev), -1)
    e = R.rounded(e, s, dx.dtype)
    bx = R.product_bound(s, w.double(), e, 2 * d)
    R.assert_within(dx, want_x, R.rounded(bx, want_x, dx.dtype), label + " dx")
    bw = R.product_bound(s.T, x.double(), e.T, x.shape[0])
    R.assert_within(dw, want_w, R.rounded(bw, want_w, dw.dtype), label + " dw")
    # Two roundings, S's and the output's.
    R.assert_near(dx, want_x, R.rounding_noise(s, w.double(), dx.dtype), label + " dx")
    R.assert_near(dw, want_w, R.rounding_noise(s.T, x.double(), dx.dtype), label + " dw")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(cuda, shape, dt):
    rows, hidden, d = shape
    act = ("silu", "gelu", "gelu_tanh")[(rows + d) % 3]
    x, w, dout = make(rows, hidden, d, DTYPES[dt], cuda)
    gate_up = torch.full((rows, 2 * d), float("nan"), device=cuda)
    out = hp.gated_linear(x, w, act, gate_up=gate_up)
    assert torch.equal(out, hp.gated_linear(x, w, act))
    check_forward(out, x, w, act, f"{shape} {dt} {act}")
    gu = (x.double() @ w.double().T)
    R.assert_within(gate_up, gu, hidden * R.F32 * (x.double().abs() @ w.double().abs().T) + 1e-30, "gate_up")
    kept = hp.gated_linear_backward(dout, x, w, act, gate_up=gate_up)
    again = hp.gated_linear_backward(dout, x, w, act)
    for (dx, dw), how in ((kept, "kept"), (again, "again")):
        check_backward(dx, dw, dout, x, w, act, f"{shape} {dt} {act} {how}")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_every_activation(cuda, act, dt):
    x, w, dout = make(40, 128, 96, DTYPES[dt], cuda)
    x *= 4  # gates up to about 16: both saturated ends
    check_forward(hp.gated_linear(x, w, act), x, w, act, act)
    check_backward(*hp.gated_linear_backward(dout, x, w, act), dout, x, w, act, act)


@pytest.mark.parametrize("pad", [1, 8, 24])
def test_strided_rows_and_views(cuda, pad):
    """Rows that are slices of wider buffers, the weight's and the outputs' among them."""
    rows, hidden, d = 70, 136, 104
    x, w, dout = make(rows, hidden, d, torch.bfloat16, cuda, pad=pad)
    wide = torch.zeros(2 * d, hidden + pad, dtype=w.dtype, device=cuda)
    wide[:, pad:] = w
    out = torch.full((rows, d + pad), 7.0, dtype=w.dtype, device=cuda)
    gate_up = torch.full((rows, 2 * d + pad), 7.0, device=cuda)
    got = hp.gated_linear(x, wide[:, pad:], "silu", out=out[:, :d], gate_up=gate_up[:, :2 * d])
    check_forward(got, x, w, "silu", f"pad {pad}")
    assert (out[:, d:] == 7).all() and (gate_up[:, 2 * d:] == 7).all()
    got = hp.gated_linear_backward(dout, x, wide[:, pad:], "silu", gate_up=gate_up[:, :2 * d])
    check_backward(*got, dout, x, w, "silu", f"pad {pad}")


def test_leading_dimensions_and_empty(cuda):
    x, w, dout = make(12, 64, 48, torch.float16, cuda)
    out = hp.gated_linear(x.view(3, 4, 64), w)
    assert out.shape == (3, 4, 48) and torch.equal(out.view(12, 48), hp.gated_linear(x, w))
    dx, dw = hp.gated_linear_backward(dout.view(3, 4, 48), x.view(3, 4, 64), w)
    assert dx.shape == (3, 4, 64) and torch.equal(dw, hp.gated_linear_backward(dout, x, w)[1])
    assert hp.gated_linear(x[:0], w).shape == (0, 48)
    dx, dw = hp.gated_linear_backward(dout[:0], x[:0], w)
    assert dx.shape == (0, 64) and not dw.any()
    dx, dw = hp.gated_linear_backward(dout[:, :0], x, w[:0])
    assert not dx.any() and dw.shape == (0, 64)
    assert not hp.gated_linear(x[:, :0], w[:, :0]).any()


def test_infinities_stay_in_their_rows(cuda):
    x, w, _ = make(130, 64, 72, torch.bfloat16, cuda)
    clean = hp.gated_linear(x, w)
    x[5, 3], x[129, 0] = float("inf"), float("nan")
    out = hp.gated_linear(x, w)
    keep = torch.ones(130, dtype=torch.bool, device=cuda)
    keep[5] = keep[129] = False
    assert torch.equal(out[keep], clean[keep]) and out[129].isnan().all()


def test_streams_and_graphs(cuda):
    x, w, dout = make(65, 256, 160, torch.bfloat16, cuda)
    want = (hp.gated_linear(x, w), *hp.gated_linear_backward(dout, x, w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = (hp.gated_linear(x, w), *hp.gated_linear_backward(dout, x, w))
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = (hp.gated_linear(x, w), *hp.gated_linear_backward(dout, x, w))
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, kept):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_no_wait_gave_up(cuda):
    """The products' and the norm's backward kernels wait with a limit; none may run out."""
    import ctypes

    from hp_rms_norm_b200 import capi

    x, w, dout = make(700, 192, 130, torch.bfloat16, cuda)
    hp.gated_linear(x, w)
    hp.gated_linear_backward(dout, x, w)
    hp.rms_norm_backward(x, x, x[0].contiguous(), 1e-6)
    t = torch.zeros(700, dtype=torch.int64, device=cuda)
    hp.linear_cross_entropy(x, w, t)
    torch.cuda.synchronize()
    count = ctypes.c_uint(7)
    assert capi.load().hprn_wait_timeouts(ctypes.byref(count), 0) == 0 and count.value == 0


@pytest.mark.parametrize("rows", [600, 2100])
def test_unaligned_rows_in_large_products(cuda, rows):
    """Operands that are copied to aligned rows, and outputs on odd addresses."""
    x, w, dout = make(rows, 129, 140, torch.float16, cuda)
    check_forward(hp.gated_linear(x, w), x, w, "silu", f"{rows}")
    check_backward(*hp.gated_linear_backward(dout, x, w), dout, x, w, "silu", f"{rows}")
    x, w, dout = make(rows, 136, 140, torch.bfloat16, cuda)  # 16-byte rows inside 32-byte sectors
    check_forward(hp.gated_linear(x, w), x, w, "silu", f"{rows}")
    check_backward(*hp.gated_linear_backward(dout, x, w), dout, x, w, "silu", f"{rows}")


def test_refusals(cuda):
    x, w, dout = make(4, 32, 16, torch.bfloat16, cuda)
    for bad in (lambda: hp.gated_linear(x.cpu(), w), lambda: hp.gated_linear(x, w.half()),
                lambda: hp.gated_linear(x.float(), w.float()), lambda: hp.gated_linear(x, w, "relu"),
                lambda: hp.gated_linear(x, w[:-1]), lambda: hp.gated_linear(x[:, :-1], w),
                lambda: hp.gated_linear(x, w, out=torch.empty(4, 15, dtype=x.dtype, device=cuda)),
                lambda: hp.gated_linear(x, w, out=x[:, :16]),
                lambda: hp.gated_linear(x, w, gate_up=torch.empty(4, 32, dtype=x.dtype, device=cuda)),
                lambda: hp.gated_linear(x.t().contiguous().t(), w),
                lambda: hp.gated_linear_backward(dout[:3], x, w),
                lambda: hp.gated_linear_backward(dout.half(), x, w),
                lambda: hp.gated_linear_backward(dout, x, w, gate_up=torch.empty(4, 16, device=cuda))):
        with pytest.raises(RuntimeError):
            bad()
