"""linear_log_probs and its backward pass on the GPU against the 64-bit formulas."""
import ctypes
import math

import pytest
import torch

import hp_rms_norm_b200 as hp
from tests import block_reference as B
from tests import training_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100
SHAPES = [(1, 64, 256), (1, 1001, 1), (2, 8, 3), (7, 1, 31), (9, 264, 1000), (33, 40, 513),
          (64, 512, 2048), (100, 1000, 333), (129, 136, 4097), (300, 520, 1500), (513, 264, 777)]


def make(rows, hidden, vocab, dtype, device, ignored=0.2, scale=2.0, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + rows * 7 + hidden * 3 + vocab)
    x = torch.randn(rows, hidden, generator=g, device=device).to(dtype)
    w = (torch.randn(vocab, hidden, generator=g, device=device) * scale * hidden ** -0.5).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    t[torch.rand(rows, generator=g, device=device) < ignored] = IGNORE
    c = torch.randn(rows, generator=g, device=device)
    h = torch.rand(rows, generator=g, device=device) * 0.5
    return x, w, t, c, h


def ranked(logits, top):
    """The largest ones, equal ones by their indices."""
    value, order = logits.sort(dim=-1, descending=True, stable=True)
    return value[:, :top], order[:, :top]


def check_forward(found, x, w, t, temperature, top, label):
    log_prob, entropy, lse, logits = B.log_probs(x, w, t, IGNORE, temperature)
    each, lse_err, entropy_err = B.log_prob_errors(x, w, temperature)
    counts = (t != IGNORE).double()
    e = each.max(-1).values
    R.assert_within(found.lse, lse, lse_err, label + " lse")
    R.assert_within(found.log_prob, log_prob, (lse_err + e + 2 * R.F32 * (log_prob.abs() + lse.abs())) * counts, label + " log_prob")
    R.assert_within(found.entropy, entropy, entropy_err * counts, label + " entropy")
    if not top:
        assert found.top_log_probs is None and found.top_indices is None
        return
    value, order = ranked(logits, top)
    assert torch.equal(found.top_indices, order), label
    want = value - lse[:, None]
    # The values come from logits in 64 bits; only lse and the rounding to fp32 are off.
    R.assert_within(found.top_log_probs, want, lse_err[:, None] + R.F32 * (want.abs() + 1e-30), label + " top")


def check_backward(grads, c, x, w, t, temperature, h, label):
    dx, dw = grads
    want_x, want_w, s, err = B.log_probs_backward(c, x, w, t, IGNORE, temperature, h)
    u = R.U[dx.dtype]
    # fp16 holds S times 2^13 or more over the largest gradient; below its smallest normal it is off by 2^-25.
    most = max(float(c.abs().max()), 0.0 if h is None else float(h.abs().max()))
    tiny = R.TINY[dx.dtype] * (most * 2.0 ** -13 / temperature if dx.dtype == torch.float16 else 1.0)
    e = err + u * (s.abs() + err) + tiny
    bx = R.product_bound(s, w.double(), e, w.shape[0])
    R.assert_within(dx, want_x, R.rounded(bx, want_x, dx.dtype), label + " dx")
    bw = R.product_bound(s.T, x.double(), e.T, x.shape[0])
    R.assert_within(dw, want_w, R.rounded(bw, want_w, dw.dtype), label + " dw")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(cuda, shape, dt):
    x, w, t, c, h = make(*shape, DTYPES[dt], cuda)
    for temperature, top, entropy in ((1.0, 0, None), (0.7, min(5, shape[2]), h)):
        found = hp.linear_log_probs(x, w, t, top=top, temperature=temperature)
        label = f"{shape} {dt} at {temperature}"
        check_forward(found, x, w, t, temperature, top, label)
        grads = hp.linear_log_probs_backward(c, x, w, t, found.lse, entropy=found.entropy, grad_entropy=entropy, temperature=temperature)
        check_backward(grads, c, x, w, t, temperature, entropy, label)


@pytest.mark.parametrize("top", [1, 2, 20, 64])
@pytest.mark.parametrize("shape", [(1, 64, 64), (5, 72, 65), (40, 128, 5000), (3, 33, 40001)], ids=str)
def test_alternatives(cuda, shape, top):
    x, w, t, _, _ = make(*shape, torch.bfloat16, cuda)
    check_forward(hp.linear_log_probs(x, w, t, top=top), x, w, t, 1.0, top, f"{shape} top {top}")


def test_equal_logits_go_to_the_lowest_index(cuda):
    """Weights with equal rows, a whole vocabulary of them, and inputs of zeros."""
    x, w, t, _, _ = make(70, 96, 3000, torch.bfloat16, cuda)
    w[1500:] = w[:1500]
    x[3] = 0
    x[64:] = 0
    check_forward(hp.linear_log_probs(x, w, t, top=10), x, w, t, 1.0, 10, "pairs")
    w[:] = w[7]
    found = hp.linear_log_probs(x, w, t, top=33)
    assert torch.equal(found.top_indices, torch.arange(33, device=cuda).expand(70, 33))
    assert (found.top_log_probs == found.top_log_probs[:, :1]).all()


def test_neighbours_in_the_last_bits(cuda):
    """Logits that differ by less than the rounding of an fp32 sum are ordered as in 64 bits: columns
    whose weights differ in one element that meets an input of 2^-20."""
    g = torch.Generator(device=cuda).manual_seed(5)
    x, w, t, _, _ = make(32, 512, 2000, torch.bfloat16, cuda)
    x[:, 100] = 2.0 ** -20
    for k in range(0, 2000, 2):
        w[k + 1] = w[k]
    w[:, 100] = torch.randint(-64, 65, (2000,), generator=g, device=cuda).to(w.dtype) / 64
    _, order = ranked(x.double() @ w.double().T, 12)
    assert torch.equal(hp.linear_log_probs(x, w, t, top=12).top_indices, order)


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("rows,vocab", [(1, 300), (8, 5000), (64, 5000), (300, 40001)], ids=str)
def test_rows_whose_largest_has_the_weight(cuda, rows, vocab, temperature):
    """No alternative's value is above 0, in rows with nearly all weight on one token, rows that are
    flat, rows of zeros.  Where one has all of it but 2^-30, its value is 0 to 2^-23, whatever the
    rounding of lse, and so is its log probability."""
    x, w, _, _, _ = make(rows, 128, vocab, torch.bfloat16, cuda, scale=20.0)
    x[rows // 2] = 0
    x[:rows // 3] /= 16
    x[-1] = 4 * w[7]
    logits = x.double() @ w.double().T / temperature
    best = logits.topk(2, dim=-1)
    # The others are at most vocab - 1 times the second.
    sharp = best.values[:, 0] - best.values[:, 1] > 21 + math.log(vocab)
    assert sharp.any()
    found = hp.linear_log_probs(x, w, best.indices[:, 0].contiguous(), top=5, temperature=temperature)
    assert torch.equal(found.top_indices[sharp, 0], best.indices[sharp, 0])
    assert (found.top_log_probs <= 0).all()
    assert (found.top_log_probs[sharp, 0] >= -(2.0 ** -23)).all() and (found.log_prob[sharp].abs() <= 2.0 ** -23).all()


def test_blocks_of_rows(cuda):
    """A vocabulary whose logits fill the workspace with 1 GiB: several blocks of rows."""
    rows, vocab = 700, 600001
    x, w, t, _, _ = make(rows, 24, vocab, torch.float16, cuda)
    found = hp.linear_log_probs(x, w, t, top=7)
    for k in (slice(0, 40), slice(250, 262), slice(440, 452), slice(690, 700)):
        part = hp.LogProbs(*(None if v is None else v[k] for v in found))
        check_forward(part, x[k], w, t[k], 1.0, 7, f"rows {k}")


@pytest.mark.parametrize("vocab", [33, 70, 257, 600, 1500, 4001, 8160, 8192, 8200])
def test_few_groups(cuda, vocab):
    """Vocabularies of fewer groups of 32 than threads search them, after a call whose logits are
    larger, so that what a CTA finds in shared memory is of no use."""
    big = make(500, 64, 40000, torch.bfloat16, cuda, scale=50.0)
    for rows in (5, 300):
        x, w, t, _, _ = make(rows, 64, vocab, torch.bfloat16, cuda)
        for top in (1, 3, 20, min(vocab, 64)):
            hp.linear_log_probs(*big[:3], top=20)
            check_forward(hp.linear_log_probs(x, w, t, top=top), x, w, t, 1.0, top, f"{rows} x {vocab} top {top}")


@pytest.mark.parametrize("rows,vocab,top", [(2600, 20003, 1), (2601, 20003, 5), (300, 90001, 20), (19000, 10300, 1)])
def test_many_rows_of_a_long_vocabulary(cuda, rows, vocab, top):
    """Rows and vocabularies large enough that a first part of the columns tells which logits of the
    others matter; the largest ones in the first part, in the last, equal in both, and one value."""
    x, w, t, _, _ = make(rows, 40, vocab, torch.bfloat16, cuda)
    w[-700:-350] = w[:350]
    w[:, 39] = 0
    x[:, 39] = 8
    w[:64, 39] = (torch.arange(64, device=cuda) % 8).to(w.dtype)
    w[-64:, 39] = (torch.arange(64, device=cuda) % 16).to(w.dtype)
    x[:50, 39] = -8
    x[50:60] = 0
    found = hp.linear_log_probs(x, w, t, top=top)
    x64 = torch.cat([x[:120], x[-120:]])
    part = hp.LogProbs(*(None if v is None else torch.cat([v[:120], v[-120:]]) for v in found))
    check_forward(part, x64, w, torch.cat([t[:120], t[-120:]]), 1.0, top, f"{rows} rows, {top}")
    x[7] = float("nan")
    x[8, 3] = float("inf")
    again = hp.linear_log_probs(x, w, t, top=top)
    assert again.top_log_probs[7:9].isnan().all()
    for a, b in zip(found, again):
        assert torch.equal(a[9:], b[9:]) and torch.equal(a[:7], b[:7])


@pytest.mark.parametrize("dt", list(DTYPES))
def test_sharp_and_flat_logits(cuda, dt):
    """Logits of several hundred, where nearly all probability is one token's, and equal ones."""
    x, w, t, c, h = make(70, 128, 600, DTYPES[dt], cuda, scale=60.0)
    found = hp.linear_log_probs(x, w, t, top=3)
    check_forward(found, x, w, t, 1.0, 3, "sharp")
    check_backward(hp.linear_log_probs_backward(c, x, w, t, found.lse, found.entropy, h), c, x, w, t, 1.0, h, "sharp")
    found = hp.linear_log_probs(x * 0, w, t)
    counted = found.entropy[t != IGNORE]
    assert (counted - torch.tensor(600.0).log().item()).abs().max() <= 4 * R.F32 * 7


def test_small_temperatures(cuda):
    x, w, t, c, h = make(65, 128, 900, torch.bfloat16, cuda)
    for temperature in (0.05, 3.0, 50.0):
        found = hp.linear_log_probs(x, w, t, top=4, temperature=temperature)
        check_forward(found, x, w, t, temperature, 4, f"at {temperature}")
        grads = hp.linear_log_probs_backward(c, x, w, t, found.lse, found.entropy, h, temperature=temperature)
        check_backward(grads, c, x, w, t, temperature, h, f"at {temperature}")


def test_same_as_the_loss(cuda):
    x, w, t, c, _ = make(200, 264, 3001, torch.bfloat16, cuda)
    loss, lse = hp.linear_cross_entropy(x, w, t)
    found = hp.linear_log_probs(x, w, t)
    torch.testing.assert_close(found.log_prob, -loss, rtol=4 * R.F32, atol=8 * R.F32 * 12)
    torch.testing.assert_close(found.lse, lse, rtol=4 * R.F32, atol=0)
    for a, b in zip(hp.linear_cross_entropy_backward(c, x, w, t, lse), hp.linear_log_probs_backward(-c, x, w, t, lse)):
        assert torch.equal(a, b)


def test_ignored_and_invalid_rows(cuda):
    x, w, t, c, h = make(130, 64, 300, torch.bfloat16, cuda, ignored=0.0)
    t[:] = IGNORE
    c[3], h[4] = float("inf"), float("nan")
    x[5] = float("nan")
    found = hp.linear_log_probs(x, w, t, top=2)
    assert not found.log_prob.any() and not found.entropy.any()
    assert ((found.top_indices >= 0) & (found.top_indices < 300)).all()
    dx, dw = hp.linear_log_probs_backward(c, x, w, t, found.lse, found.entropy, h)
    assert not dx.any() and not dw.any()
    x[5], c[3], h[4] = 0, 1, 1
    t[:] = 5
    t[0], t[129], t[7], t[8] = 299, 0, 300, -1
    found = hp.linear_log_probs(x, w, t)
    assert found.log_prob[[7, 8]].isnan().all() and torch.isfinite(found.log_prob).sum() == 128
    dx, _ = hp.linear_log_probs_backward(c, x, w, t, found.lse, found.entropy, h)
    assert dx[[7, 8]].isnan().all() and torch.isfinite(dx).all(-1).sum() == 128


def test_infinite_weights(cuda):
    """Logits of -inf have probability 0 and add nothing to the entropy; a NaN row is its own."""
    x, w, t, _, _ = make(40, 64, 500, torch.bfloat16, cuda, ignored=0.0)
    x = x.abs() + 0.5
    t[:] = 3
    want = hp.linear_log_probs(x, w[:400], t)
    w[400:, 0] = float("-inf")
    found = hp.linear_log_probs(x, w, t, top=6)
    torch.testing.assert_close(found.entropy, want.entropy, rtol=1e-5, atol=0)
    torch.testing.assert_close(found.log_prob, want.log_prob, rtol=1e-5, atol=0)
    assert (found.top_indices < 400).all()
    x[11, 5] = float("nan")
    found = hp.linear_log_probs(x, w, t, top=6)
    assert found.log_prob[11].isnan() and found.entropy[11].isnan() and torch.isfinite(found.entropy).sum() == 39
    assert ((found.top_indices >= 0) & (found.top_indices < 500)).all()


def test_empty(cuda):
    x, w, t, c, h = make(12, 64, 48, torch.float16, cuda)
    found = hp.linear_log_probs(x[:0], w, t[:0], top=3)
    assert found.log_prob.shape == (0,) and found.top_indices.shape == (0, 3)
    dx, dw = hp.linear_log_probs_backward(c[:0], x[:0], w, t[:0], found.lse)
    assert dx.shape == (0, 64) and not dw.any()
    found = hp.linear_log_probs(x, w[:0], torch.full_like(t, IGNORE))
    assert not found.log_prob.any() and not found.entropy.any() and (found.lse == float("-inf")).all()
    found = hp.linear_log_probs(x[:, :0], w[:, :0], t, top=2)
    torch.testing.assert_close(found.lse, torch.full_like(found.lse, 48.0).log())
    assert torch.equal(found.top_indices, torch.arange(2, device=cuda).expand(12, 2))


def test_strides(cuda):
    x, w, t, c, h = make(50, 200, 700, torch.bfloat16, cuda)
    wide_x, wide_w = torch.zeros(50, 211, dtype=x.dtype, device=cuda), torch.zeros(700, 203, dtype=x.dtype, device=cuda)
    wide_x[:, 3:203], wide_w[:, 1:201] = x, w
    want = hp.linear_log_probs(x, w, t, top=4)
    got = hp.linear_log_probs(wide_x[:, 3:203], wide_w[:, 1:201], t, top=4)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_pieces_of_the_vocabulary(cuda):
    rows, vocab = 40000, 9001
    x, w, t, c, h = make(rows, 16, vocab, torch.bfloat16, cuda)
    t[0], t[1], t[2] = 0, vocab - 1, 6400
    found = hp.linear_log_probs(x, w, t)
    dx, dw = hp.linear_log_probs_backward(c, x, w, t, found.lse, found.entropy, h)
    want_x, want_w, s, _ = B.log_probs_backward(c, x, w, t, IGNORE, 1.0, h)
    R.assert_near(dx, want_x, R.rounding_noise(s, w.double(), w.dtype), "dx")
    R.assert_near(dw, want_w, R.rounding_noise(s.T, x.double(), w.dtype), "dw")


def test_differences(cuda):
    """The operator's own differences in random directions; inputs and steps exact in bf16, as in
    the cross entropy's test."""
    g = torch.Generator(device=cuda).manual_seed(1)
    rows, hidden, vocab = 48, 64, 400
    x = (torch.randint(-12, 13, (rows, hidden), generator=g, device=cuda) / 16).bfloat16()
    w = (torch.randint(-12, 13, (vocab, hidden), generator=g, device=cuda) / 32).bfloat16()
    t = torch.randint(0, vocab, (rows,), generator=g, device=cuda)
    c, k = 1.0, 0.5
    found = hp.linear_log_probs(x, w, t)
    dx, _ = hp.linear_log_probs_backward(torch.full((rows,), c, device=cuda), x, w, t, found.lse, found.entropy,
                                         torch.full((rows,), k, device=cuda))

    def value(v):
        f = hp.linear_log_probs(v.bfloat16(), w, t)
        return c * f.log_prob.double() + k * f.entropy.double()

    h = 2.0 ** -5
    for _ in range(4):
        v = (torch.randint(0, 2, x.shape, generator=g, device=cuda) * 2 - 1).double()
        diff = (value(x.double() + h * v) - value(x.double() - h * v)) / (2 * h)
        along = (dx.double() * v).sum(-1)
        # With L(h) = L + h u the third derivatives are central moments of u under p, times log p for the
        # entropy: at most |u|^3 times 2 for the log probability, and 2 (|log p| + 7) + 14 for the entropy.
        u = (w.double() @ v.T).abs().max(0).values
        log_p = 7 + 2 * (w.double() @ x.double().T).abs().max(0).values
        third = h * h / 6 * u ** 3 * (2 * c + k * (2 * (log_p + 7) + 14))
        bound = third + 2 * 14 * 8 * R.F32 / h + 3 * R.U[torch.bfloat16] * (dx.double().abs().sum(-1) + (c + 4 * k) * 0.4)
        assert ((diff - along).abs() <= bound).all()


def test_autograd(cuda):
    from hp_rms_norm_b200 import autograd as A

    x, w, t, c, h = make(66, 128, 500, torch.bfloat16, cuda)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    log_prob, entropy = A.linear_log_probs(a, b, t, temperature=0.8)
    found = hp.linear_log_probs(x, w, t, temperature=0.8)
    assert torch.equal(log_prob, found.log_prob) and torch.equal(entropy, found.entropy)
    for outs, grads, args in (((log_prob, entropy), (c, h), (c, h)), ((log_prob,), (c,), (c, None)), ((entropy,), (h,), (c * 0, h))):
        got = torch.autograd.grad(outs, (a, b), grads, retain_graph=True)
        want = hp.linear_log_probs_backward(args[0], x, w, t, found.lse, found.entropy, args[1], temperature=0.8)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_streams_graphs_and_shapes(cuda):
    x, w, t, c, h = make(66, 256, 500, torch.bfloat16, cuda)

    def both():
        f = hp.linear_log_probs(x, w, t, top=5)
        return tuple(f) + hp.linear_log_probs_backward(c, x, w, t, f.lse, f.entropy, h)

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
    f = hp.linear_log_probs(x.view(6, 11, 256), w, t.view(6, 11), top=5)
    assert f.top_indices.shape == (6, 11, 5) and torch.equal(f.top_indices.view(66, 5), want[4])


def test_refusals(cuda):
    x, w, t, c, h = make(4, 32, 16, torch.bfloat16, cuda)
    lse = torch.zeros(4, device=cuda)
    for bad in (lambda: hp.linear_log_probs(x.cpu(), w, t),
                lambda: hp.linear_log_probs(x, w.half(), t),
                lambda: hp.linear_log_probs(x, w, t.int()),
                lambda: hp.linear_log_probs(x, w, t[:3]),
                lambda: hp.linear_log_probs(x, w, t, top=17),
                lambda: hp.linear_log_probs(x, torch.cat([w] * 8), t, top=65),
                lambda: hp.linear_log_probs(x, w, t, top=-1),
                lambda: hp.linear_log_probs(x, w, t, temperature=0.0),
                lambda: hp.linear_log_probs(x, w, t, temperature=float("nan")),
                lambda: hp.linear_log_probs_backward(c.double(), x, w, t, lse),
                lambda: hp.linear_log_probs_backward(c, x, w, t, lse, temperature=-1.0),
                lambda: hp.linear_log_probs_backward(c, x, w, t, lse, grad_entropy=h),
                lambda: hp.linear_log_probs_backward(c, x, w, t, lse, entropy=lse, grad_entropy=h[:2])):
        with pytest.raises(RuntimeError):
            bad()


def test_no_wait_gave_up(cuda):
    from hp_rms_norm_b200 import capi

    torch.cuda.synchronize()
    count = ctypes.c_uint(7)
    assert capi.load().hprn_wait_timeouts(ctypes.byref(count), 0) == 0 and count.value == 0
