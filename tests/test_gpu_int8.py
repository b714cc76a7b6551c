"""rms_norm_int8, quantize_int8 and linear_int8 on the GPU against the 64-bit formulas."""
import ctypes

import pytest
import torch

import hp_rms_norm_b200 as hp
from tests import block_reference as B
from tests import training_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
ROWS = [(1, 1), (3, 7), (5, 32), (40, 250), (33, 1001), (1, 4096), (70, 1024), (9, 5001), (150, 8192), (5, 16384),
        (3, 16383), (2, 20000), (2, 33001), (3000, 1001), (700, 5001),
        (400, 12288), (3, 10240)]
# (rows, hidden, channels)
PRODUCTS = [(1, 1, 1), (1, 16, 32), (2, 15, 7), (3, 32, 64), (7, 33, 100), (16, 4096, 512), (1, 8192, 100), (33, 128, 129),
            (128, 256, 256), (130, 160, 1001), (257, 1000, 333), (300, 2731, 520), (520, 512, 1500), (1, 131071, 40),
            (3, 1000, 200), (16, 4104, 700), (1, 8, 5), (40, 5003, 3000)]


def codes(shape, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + sum(shape))
    return torch.randint(-127, 128, shape, generator=g, device=device, dtype=torch.int8)


def scales(n, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + n)
    return torch.rand(n, generator=g, device=device) * 0.02 + 0.001


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", PRODUCTS, ids=str)
def test_products(cuda, shape, dt):
    rows, hidden, channels = shape
    x, w = codes((rows, hidden), cuda), codes((channels, hidden), cuda, 1)
    xs, ws = scales(rows, cuda), scales(channels, cuda, 1)
    for bias in (None, torch.randn(channels, device=cuda).to(DTYPES[dt])):
        out = hp.linear_int8(x, xs, w, ws, bias=bias, dtype=DTYPES[dt])
        check_product(out, x, xs, w, ws, bias, f"{shape} {dt}")


def check_product(out, x, xs, w, ws, bias, label):
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    bound = 3 * R.F32 * want.abs()
    if bias is not None:
        want = want + bias.double()
        bound = bound + R.F32 * want.abs()
    # What leaves the type's range is infinite.
    inside = want.abs() < 0.999 * torch.finfo(out.dtype).max
    R.assert_within(torch.where(inside, out, 0), torch.where(inside, want, 0.0), R.rounded(bound, want, out.dtype), label)


def test_sums_are_exact(cuda):
    """The extremes: the largest sums of both signs, and scales of powers of two, so that the result is
    the sum itself rounded to fp32 and to 16 bits."""
    hidden = 131071
    x = torch.full((3, hidden), -128, dtype=torch.int8, device=cuda)
    x[1] = 127
    x[2, ::2] = 127
    w = torch.full((70, hidden), -128, dtype=torch.int8, device=cuda)
    w[1::2] = 127
    one = torch.full((3,), 2.0 ** -10, device=cuda)
    ws = torch.full((70,), 2.0 ** -10, device=cuda)
    out = hp.linear_int8(x, one, w, ws, dtype=torch.bfloat16)
    want = (x.double() @ w.double().T).float() * 2.0 ** -20
    assert torch.equal(out, want.bfloat16())
    # A row of the weight that picks one code: each code of x comes back.
    x = torch.arange(-128, 128, device=cuda).to(torch.int8).repeat(64, 1)
    pick = torch.eye(256, device=cuda).to(torch.int8)
    out = hp.linear_int8(x, torch.ones(64, device=cuda), pick, torch.ones(256, device=cuda), dtype=torch.float16)
    assert torch.equal(out, x.half())


def test_product_strides(cuda):
    rows, hidden, channels = 65, 200, 130
    x, w = codes((rows, hidden + 24), cuda), codes((channels, hidden + 16), cuda, 1)
    xs, ws = scales(rows, cuda), scales(channels, cuda, 1)
    for ox, ow in ((0, 0), (16, 0), (3, 1), (0, 5), (8, 16)):
        a, b = x[:, ox:ox + hidden], w[:, ow:ow + hidden]
        wide = torch.full((rows, channels + 9), 3.0, dtype=torch.bfloat16, device=cuda)
        hp.linear_int8(a, xs, b, ws, out=wide[:, 4:4 + channels])
        check_product(wide[:, 4:4 + channels], a, xs, b, ws, None, f"offsets {ox} {ow}")
        assert (wide[:, :4] == 3).all() and (wide[:, 4 + channels:] == 3).all()


def test_product_of_nothing(cuda):
    x, w, xs, ws = codes((4, 8), cuda), codes((6, 8), cuda), scales(4, cuda), scales(6, cuda)
    assert hp.linear_int8(x[:0], xs[:0], w, ws).shape == (0, 6)
    assert hp.linear_int8(x, xs, w[:0], ws[:0]).shape == (4, 0)
    bias = torch.arange(6, device=cuda).bfloat16()
    assert torch.equal(hp.linear_int8(x[:, :0], xs, w[:, :0], ws, bias=bias), bias.expand(4, 6))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", ROWS, ids=str)
def test_quantised_norm(cuda, shape, dt):
    rows, hidden = shape
    g = torch.Generator(device=cuda).manual_seed(rows + hidden)
    x, r = (torch.randn(rows, hidden, generator=g, device=cuda).to(DTYPES[dt]) for _ in range(2))
    w = (1 + 0.2 * torch.randn(hidden, generator=g, device=cuda)).to(DTYPES[dt])
    for residual, weight in ((None, w), (r, w), (r, None)):
        total = None if residual is None else torch.empty_like(r)
        codes, scale = hp.rms_norm_int8(x, weight, EPS, residual=residual, residual_out=total)
        y, err, want_total = B.rms_norm_int8(x, weight, EPS, residual)
        most = y.abs().amax(-1)
        worst = (err / y.abs().clamp(min=1e-30)).max()
        R.assert_within(scale, most.clamp(min=1e-12) / 127, (worst + 2 * R.F32) * most / 127 + 1e-20, f"{shape} scale")
        assert codes.abs().max() <= 127
        # Half a step, and what fp32 operations may move y / scale by.
        off = (codes.double() - y * 127 / most.clamp(min=1e-12)[:, None]).abs()
        assert (off <= 0.5 + 127 * (2 * worst + 4 * R.F32)).all()
        if residual is not None:
            assert torch.equal(total, (x.float() + r.float()).to(x.dtype))
            again = r.clone()
            codes2, scale2 = hp.rms_norm_int8(x, weight, EPS, residual=again)
            assert torch.equal(codes, codes2) and torch.equal(scale, scale2) and torch.equal(again, total)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", ROWS, ids=str)
def test_quantise(cuda, shape, dt):
    """fp32 operations in the documented order: the same bits."""
    x = torch.randn(*shape, device=cuda).to(DTYPES[dt])
    x[0] = 0
    codes, scale = hp.quantize_int8(x)
    want_scale = x.float().abs().amax(-1).clamp(min=1e-12) / torch.tensor(127.0, device=cuda)
    assert torch.equal(scale, want_scale)
    want = torch.round(x.float() * (torch.ones_like(scale) / scale)[:, None])
    assert torch.equal(codes, want.to(torch.int8))


def test_quantised_strides_and_values(cuda):
    wide = torch.randn(40, 600, device=cuda).bfloat16()
    for offset, hidden in ((0, 512), (1, 511), (8, 520), (4, 300)):
        x = wide[:, offset:offset + hidden]
        out = torch.full((40, hidden + 40), 55, dtype=torch.int8, device=cuda)
        scale = torch.empty(40, device=cuda)
        torch.ops.hp_rms_norm.rms_norm_int8.out(out[:, 8:8 + hidden], scale, x, None, None, None, 0.0)
        want, want_scale = hp.quantize_int8(x.contiguous())
        assert torch.equal(out[:, 8:8 + hidden], want) and torch.equal(scale, want_scale)
        assert (out[:, :8] == 55).all() and (out[:, 8 + hidden:] == 55).all()
    x = wide[:4, :64].clone()
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    codes, scale = hp.quantize_int8(x)
    assert scale[1].isnan() and scale[2].isinf() and torch.isfinite(scale[[0, 3]]).all()
    y = hp.linear_int8(codes, scale, torch.ones(32, 64, dtype=torch.int8, device=cuda), torch.ones(32, device=cuda))
    assert y[1:3].isnan().all() and torch.isfinite(y[[0, 3]]).all()


def test_streams_and_graphs(cuda):
    x, w, ws = torch.randn(70, 520, device=cuda).half(), codes((300, 520), cuda), scales(300, cuda)
    weight = torch.ones(520, device=cuda).half()

    def both():
        q, s = hp.rms_norm_int8(x, weight, EPS)
        return q, s, hp.linear_int8(q, s, w, ws, dtype=torch.float16), hp.linear_int8(q[:, :333], s, w[:, 1:334], ws, dtype=torch.float16)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    graphs, kept = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept.append(both())
        graphs.append(g)
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for a, b, p, q in zip(want, other, *kept):
        assert torch.equal(a, b) and torch.equal(a, p) and torch.equal(a, q)


def test_refusals(cuda):
    x, w, xs, ws = codes((4, 8), cuda), codes((6, 8), cuda), scales(4, cuda), scales(6, cuda)
    h = torch.randn(4, 8, device=cuda).half()
    big = torch.zeros(1, 131072, dtype=torch.int8, device=cuda)
    for bad in (lambda: hp.linear_int8(x.cpu(), xs, w, ws),
                lambda: hp.linear_int8(h, xs, w, ws),
                lambda: hp.linear_int8(x, xs[:3], w, ws),
                lambda: hp.linear_int8(x, xs, w, ws.double()),
                lambda: hp.linear_int8(x, xs, w[:, :7], ws),
                lambda: hp.linear_int8(x, xs, w, ws, dtype=torch.float32),
                lambda: hp.linear_int8(x, xs, w, ws, bias=torch.zeros(6, device=cuda)),
                lambda: hp.linear_int8(x, xs, w, ws, bias=torch.zeros(5, device=cuda).bfloat16()),
                lambda: hp.linear_int8(big, xs[:1], big, xs[:1]),
                lambda: hp.rms_norm_int8(h.float(), None, EPS),
                lambda: hp.rms_norm_int8(h, h[0, :7], EPS),
                lambda: hp.rms_norm_int8(h, h[0], EPS, residual=h[:2]),
                lambda: hp.rms_norm_int8(h, h[0].clone(), EPS, residual_out=h.clone()),
                lambda: hp.rms_norm_int8(h, h[0].clone(), EPS, residual=h)):
        with pytest.raises(RuntimeError):
            bad()


def test_no_wait_gave_up(cuda):
    from hp_rms_norm_b200 import capi

    torch.cuda.synchronize()
    count = ctypes.c_uint(7)
    assert capi.load().hprn_wait_timeouts(ctypes.byref(count), 0) == 0 and count.value == 0
