"""gated_add_rms_norm and its backward pass on the GPU against the 64-bit formulas."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from tests import block_reference as B
from tests import training_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
# (leading dimensions, hidden)
SHAPES = [((1,), 1), ((3,), 7), ((5,), 32), ((2, 9), 64), ((33,), 250), ((4, 17), 1001), ((1,), 4096), ((70,), 1024),
          ((12, 11), 2056), ((9,), 5001), ((150,), 8192), ((6,), 16384), ((3,), 16383), ((2,), 20000), ((2, 2), 33001),
          ((400,), 10240), ((3,), 9216), ((170, 2), 12288)]
GATES = ["none", "channel", "token", "sequence", "one for each sequence", "full", "one"]


def gate_shape(kind, lead, hidden):
    ones = (1,) * (len(lead) - 1)
    return {"none": None, "channel": (hidden,), "token": lead + (1,), "sequence": lead[:1] + ones + (hidden,),
            "one for each sequence": lead[:1] + ones + (1,), "full": lead + (hidden,), "one": (1,)}[kind]


def make(lead, hidden, dtype, device, gate="channel", post=True, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + hidden * 3 + sum(lead))

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device=device) * scale + mean).to(dtype)

    shape = gate_shape(gate, lead, hidden)
    return {"x": normal(*lead, hidden), "r": normal(*lead, hidden, scale=3.0), "p": normal(hidden, scale=0.2, mean=0.6) if post else None,
            "w": normal(hidden, scale=0.2, mean=1.0), "gate": None if shape is None else normal(*shape, mean=0.5),
            "d": normal(*lead, hidden, scale=0.3), "e": normal(*lead, hidden, scale=0.3)}


def check(s, scale, label, with_e=True):
    out, total = torch.empty_like(s["x"]), torch.empty_like(s["r"])
    got = hp.gated_add_rms_norm(s["x"], s["r"], s["p"], s["w"], EPS, gate=s["gate"], residual_scale=scale, out=out, residual_out=total)
    assert got is out
    (want, bound), (want_t, bound_t) = B.gated_add_rms_norm(s["x"], s["r"], s["p"], s["w"], EPS, s["gate"], scale)
    R.assert_within(total, want_t, R.rounded(bound_t, want_t, total.dtype), label + " residual")
    R.assert_within(out, want, R.rounded(bound, want, out.dtype), label + " out")
    e = s["e"] if with_e else None
    grads = hp.gated_add_rms_norm_backward(s["d"], s["x"], total, s["p"], s["w"], EPS, gate=s["gate"], residual_scale=scale, grad_residual=e)
    want = B.gated_add_rms_norm_backward(s["d"], s["x"], total, s["p"], s["w"], EPS, s["gate"], scale, e)
    for name, got in zip(("x", "residual", "post_weight", "weight", "gate"), grads):
        if name not in want:
            assert got is None
            continue
        value, bound = want[name]
        assert got.shape == value.shape
        R.assert_within(got, value, R.rounded(bound, value, got.dtype), f"{label} grad {name}")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(cuda, shape, dt):
    check(make(*shape, DTYPES[dt], cuda), 0.75, f"{shape} {dt}")


@pytest.mark.parametrize("post", [True, False], ids=["post", "no post"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("shape", [((7, 5), 264), ((3, 4, 5), 1001), ((40, 2), 2048), ((1, 130), 1000)], ids=str)
def test_gates(cuda, shape, gate, post):
    check(make(*shape, torch.bfloat16, cuda, gate=gate, post=post), 1.0, f"{shape} {gate}")
    check(make(*shape, torch.float16, cuda, gate=gate, post=post), 0.5, f"{shape} {gate}", with_e=False)


def test_many_rows(cuda):
    """Grids of several waves, many partial sums, gates that few rows share."""
    check(make((2500, 2), 512, torch.bfloat16, cuda, gate="sequence"), 1.0, "5000 rows, 2500 gates")
    check(make((5, 1000), 768, torch.bfloat16, cuda, gate="sequence"), 1.0, "5000 rows, 5 gates")
    check(make((5000,), 1024, torch.float16, cuda, gate="token"), 1.0, "5000 rows, a gate each")
    check(make((6, 1000), 2003, torch.float16, cuda, gate="sequence"), 0.5, "6000 odd rows")


def test_strides_and_offsets(cuda):
    for offset, pad in ((0, 8), (1, 3), (4, 20), (8, 16)):
        s = make((37,), 520, torch.bfloat16, cuda, gate="full")
        for k in ("x", "r", "gate", "d", "e"):
            wide = torch.full((37, 520 + pad + offset), float("nan"), dtype=torch.bfloat16, device=cuda)
            wide[:, offset:offset + 520] = s[k]
            s[k] = wide[:, offset:offset + 520]
        for k in ("p", "w"):
            wide = torch.full((520 + offset,), float("nan"), dtype=torch.bfloat16, device=cuda)
            wide[offset:] = s[k]
            s[k] = wide[offset:]
        check(s, 0.5, f"offset {offset} pad {pad}")


@pytest.mark.parametrize("hidden", [256, 1001, 20000])
def test_in_place_and_neighbours(cuda, hidden):
    """residual updated in place, out over input; rows around the ones given stay as they are."""
    s = make((6,), hidden, torch.float16, cuda)
    want_r = torch.empty_like(s["r"])
    want = hp.gated_add_rms_norm(s["x"], s["r"], s["p"], s["w"], EPS, gate=s["gate"], residual_out=want_r)
    x, r = torch.full((8, hidden), 7.0, dtype=torch.float16, device=cuda), torch.full((8, hidden), 7.0, dtype=torch.float16, device=cuda)
    x[1:7], r[1:7] = s["x"], s["r"]
    got = hp.gated_add_rms_norm(x[1:7], r[1:7], s["p"], s["w"], EPS, gate=s["gate"], out=x[1:7])
    assert torch.equal(got, want) and torch.equal(x[1:7], want) and torch.equal(r[1:7], want_r)
    for t in (x, r):
        assert (t[0] == 7).all() and (t[7] == 7).all()


def test_values(cuda):
    """Rows of zeros, and rows whose infinities and NaN stay in their rows."""
    s = make((64,), 512, torch.bfloat16, cuda, gate="token")
    s["x"][3], s["r"][3] = 0, 0
    s["x"][5] = 0
    clean = hp.gated_add_rms_norm(s["x"], s["r"].clone(), s["p"], s["w"], EPS, gate=s["gate"])
    assert not clean[3].any() and torch.isfinite(clean).all()
    check(s, 1.0, "rows of zeros")
    s["x"][7, 11], s["r"][9, 500], s["gate"][12] = float("nan"), float("inf"), 0
    total = torch.empty_like(s["r"])
    out = hp.gated_add_rms_norm(s["x"], s["r"], s["p"], s["w"], EPS, gate=s["gate"], residual_out=total)
    keep = torch.ones(64, dtype=torch.bool, device=cuda)
    keep[[7, 9, 12]] = False
    assert torch.equal(out[keep], clean[keep]) and out[7].isnan().all() and out[9, 500].isnan()
    assert torch.equal(total[12], s["r"][12])
    grads = hp.gated_add_rms_norm_backward(s["d"], s["x"], total, s["p"], s["w"], EPS, gate=s["gate"])
    assert torch.isfinite(grads[0][keep]).all() and torch.isfinite(grads[1][keep]).all()


def test_empty(cuda):
    s = make((4,), 64, torch.bfloat16, cuda)
    x = s["x"][:0]
    assert hp.gated_add_rms_norm(x, s["r"][:0], s["p"], s["w"], EPS, gate=s["gate"]).shape == (0, 64)
    grads = hp.gated_add_rms_norm_backward(x, x, x, s["p"], s["w"], EPS, gate=s["gate"])
    assert grads[0].shape == (0, 64) and not any(g.any() for g in grads)
    x = s["x"][:, :0]
    assert hp.gated_add_rms_norm(x, x.clone(), s["p"][:0], s["w"][:0], EPS).shape == (4, 0)


def test_differences(cuda):
    """The gradients against the operator's own differences, in 64 bits of one direction for each
    input, through the autograd form: a sum weighted by powers of two over fp32 differences."""
    from hp_rms_norm_b200 import autograd as A

    g = torch.Generator(device=cuda).manual_seed(3)
    lead, hidden = (8, 4), 96
    names = ("x", "r", "p", "w", "gate")
    s = make(lead, hidden, torch.float16, cuda, gate="sequence")
    d, e = s["d"], s["e"]
    leaves = [s[k].clone().requires_grad_() for k in names]
    out, total = A.gated_add_rms_norm(*leaves[:4], EPS, gate=leaves[4], residual_scale=0.75)
    grads = torch.autograd.grad((out, total), leaves, (d, e))

    def value(parts):
        (out, _), (total, _) = B.gated_add_rms_norm(*parts[:4], EPS, parts[4], 0.75)
        return (out * d.double()).sum() + (total * e.double()).sum()

    # The 64-bit formula's differences, to which `check` ties the kernel's forward pass.
    h = 2.0 ** -12
    for k, name in enumerate(names):
        v = torch.randn(leaves[k].shape, generator=g, device=cuda, dtype=torch.float64)
        parts = [t.detach().double() for t in leaves]
        hi, lo = list(parts), list(parts)
        hi[k], lo[k] = parts[k] + h * v, parts[k] - h * v
        diff = (value(hi) - value(lo)) / (2 * h)
        along = (grads[k].double() * v).sum()
        # Each gradient is within u of itself and, since t is read as it was rounded, within u of
        # terms of the size of |d w| inv_t; third derivatives times h^2 / 6 are below 2^-20 of that.
        size = (grads[k].double().abs() * v.abs()).sum() + (d.double().abs().sum() * 2.0 ** -4)
        assert (diff - along).abs() <= 4 * R.U[torch.float16] * size, name


def test_autograd_partial_uses(cuda):
    """Only one of the two results used; no gate, no post_weight."""
    from hp_rms_norm_b200 import autograd as A

    s = make((9,), 128, torch.bfloat16, cuda, gate="none", post=False)
    x, r, w = (s[k].clone().requires_grad_() for k in ("x", "r", "w"))
    out, total = A.gated_add_rms_norm(x, r, None, w, EPS)
    gx, gr = torch.autograd.grad(total, (x, r), s["e"], retain_graph=True)
    assert torch.equal(gx, s["e"]) and torch.equal(gr, s["e"])
    gx, gw = torch.autograd.grad(out, (x, w), s["d"])
    want = B.gated_add_rms_norm_backward(s["d"], s["x"], total.detach(), None, s["w"], EPS)
    R.assert_within(gx, want["x"][0], R.rounded(want["x"][1], want["x"][0], gx.dtype), "x")
    R.assert_within(gw, want["weight"][0], R.rounded(want["weight"][1], want["weight"][0], gw.dtype), "w")


def test_streams_and_graphs(cuda):
    s = make((6, 50), 1024, torch.bfloat16, cuda, gate="sequence")

    def both():
        total = torch.empty_like(s["r"])
        out = hp.gated_add_rms_norm(s["x"], s["r"], s["p"], s["w"], EPS, gate=s["gate"], residual_out=total)
        return (out, total) + hp.gated_add_rms_norm_backward(s["d"], s["x"], total, s["p"], s["w"], EPS, gate=s["gate"], grad_residual=s["e"])

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    graphs, kept = [], []
    for _ in range(2):  # two graphs that are replayed at once on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept.append(both())
        graphs.append(g)
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for a, b, c, d in zip(want, other, *kept):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_refusals(cuda):
    s = make((4, 3), 64, torch.bfloat16, cuda)
    x, r, p, w = s["x"], s["r"], s["p"], s["w"]
    for bad in (lambda: hp.gated_add_rms_norm(x.float(), r, p, w, EPS),
                lambda: hp.gated_add_rms_norm(x, r[:2], p, w, EPS),
                lambda: hp.gated_add_rms_norm(x, r, p[:-1], w, EPS),
                lambda: hp.gated_add_rms_norm(x, r, p, w.half(), EPS),
                lambda: hp.gated_add_rms_norm(x, r.cpu(), p, w, EPS),
                lambda: hp.gated_add_rms_norm(x, r, p, w, EPS, gate=p[:3]),
                lambda: hp.gated_add_rms_norm(x, r, p, w, EPS, gate=x[:1]),  # shared across sequences, not tokens
                lambda: hp.gated_add_rms_norm(x, r, p, w, EPS, gate=x[:, :1].expand(4, 3, 64)),
                lambda: hp.gated_add_rms_norm(x, r, p, w, EPS, gate=x[None]),
                lambda: hp.gated_add_rms_norm(x, r, p, w, EPS, out=r),
                lambda: hp.gated_add_rms_norm(x, r, p, w, EPS, residual_out=x),
                lambda: hp.gated_add_rms_norm(x, x, p, w, EPS),
                lambda: hp.gated_add_rms_norm_backward(x, x, r[:2], p, w, EPS),
                lambda: hp.gated_add_rms_norm_backward(x, x, r, p, w, EPS, gate=p[:3])):
        with pytest.raises(RuntimeError):
            bad()
