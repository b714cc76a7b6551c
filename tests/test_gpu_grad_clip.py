"""grad_norm and clip_grad_norm on the GPU against the 64-bit formulas."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from tests import training_reference as R

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(sizes, device, dtypes=TYPES, scale=1.0):
    g = torch.Generator(device=device).manual_seed(len(sizes))
    return [(scale * torch.randn(n, generator=g, device=device)).to(dtypes[k % len(dtypes)])
            for k, n in enumerate(sizes)]


def check_norm(norm, want):
    # A chunk's sum: at most 64 fp32 additions a thread and 13 more across threads,
    # of positive terms; half of that for the root.
    assert abs(norm.item() - want.item()) <= 80 * R.F32 * want.item() + 1e-30


def check_clipped(out, want, factor_error=100 * R.F32):
    for o, w in zip(out, want):
        u = R.U.get(o.dtype, 2.0 ** -24)
        tiny = R.TINY.get(o.dtype, 2.0 ** -149)
        R.assert_within(o, w, (factor_error + u) * w.abs() + tiny, "clipped")


SIZES = {"one": [1], "ragged": [5, 1, 70001, 16384, 16385, 33, 100000], "empty": [0, 10, 0],
         "many": [1 + 37 * k % 991 for k in range(1100)]}


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_norm_and_clip(cuda, name, max_norm):
    grads = make(SIZES[name], cuda)
    want_norm, want = R.clip(grads, max_norm)
    check_norm(hp.grad_norm(grads), want_norm)
    out = [torch.empty(g.shape, dtype=torch.float32, device=cuda) for g in grads]
    check_norm(hp.clip_grad_norm(grads, max_norm, out=out), want_norm)
    check_clipped(out, want)
    before = [g.clone() for g in grads]
    hp.clip_grad_norm(grads, max_norm)
    check_clipped(grads, want)
    if max_norm > 1e3:
        assert all(torch.equal(a, b) for a, b in zip(before, grads))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("to", TYPES)
def test_types_and_alignment(cuda, dtype, to):
    """Views that start at any element, in and out of step with each other."""
    flat = make([100003], cuda, [dtype])[0]
    outs = torch.empty(100010, dtype=to, device=cuda)
    at = [0, 1, 34, 4099, 20487, 60001, 100003]
    grads = [flat[a:b] for a, b in zip(at, at[1:])]
    out = [outs[a + 3:b + 3] for a, b in zip(at, at[1:])]
    want_norm, want = R.clip(grads, 2.0)
    check_norm(hp.clip_grad_norm(grads, 2.0, out=out), want_norm)
    check_clipped(out, want)


def test_layouts(cuda):
    base = torch.randn(64, 50, device=cuda)
    grads = [base[:, :30], base[:, 30:47], torch.randn(3, 5, 7, device=cuda),
             torch.tensor(2.0, device=cuda)]
    out = [torch.full((64, 30), 9.0, device=cuda), torch.full((64, 40), 9.0, device=cuda)[:, 3:20],
           torch.empty(3, 5, 7, dtype=torch.bfloat16, device=cuda), torch.empty((), device=cuda)]
    want_norm, want = R.clip(grads, 1.0)
    check_norm(hp.clip_grad_norm(grads, 1.0, out=out), want_norm)
    check_clipped(out, want)
    hp.clip_grad_norm(grads, 1.0)
    check_clipped(grads, want)


def test_non_finite(cuda):
    grads = make([1000, 20], cuda, [torch.float32])
    grads[1][3] = float("nan")
    assert hp.clip_grad_norm(grads, 1.0).isnan() and all(g.isnan().all() for g in grads)
    grads = make([1000, 20], cuda, [torch.float32])
    grads[1][3] = float("inf")
    assert hp.clip_grad_norm(grads, 1.0).isinf()
    assert grads[1][3].isnan() and not grads[0].any()
    grads = make([50], cuda, [torch.float32], scale=0.0)
    assert hp.clip_grad_norm(grads, 1.0) == 0 and not grads[0].any()
    grads = make([50], cuda, [torch.float32])
    hp.clip_grad_norm(grads, 0.0)
    assert not grads[0].any()


def test_matches_torch_utility(cuda):
    params = [torch.nn.Parameter(torch.zeros(n, device=cuda)) for n in (10, 1000, 77777)]
    for p in params:
        p.grad = torch.randn_like(p)
    ours = [p.grad.clone() for p in params]
    norm = torch.nn.utils.clip_grad_norm_(params, 3.0)
    got = hp.clip_grad_norm(ours, 3.0)
    check_norm(got, norm.double())
    check_clipped(ours, [p.grad.double() for p in params], 200 * R.F32)


def test_repeats_streams_graphs_empty(cuda):
    grads = make([70000, 3, 1 << 20], cuda)
    out = [torch.empty_like(g) for g in grads]
    norm = hp.clip_grad_norm(grads, 1.0, out=out)
    want = [o.clone() for o in out]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert hp.clip_grad_norm(grads, 1.0, out=out) == norm
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again = hp.clip_grad_norm(grads, 1.0, out=out)
    for o in out:
        o.zero_()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert again == norm and all(torch.equal(a, b) for a, b in zip(want, out))
    assert hp.clip_grad_norm([], 1.0) == 0
    assert hp.grad_norm([torch.empty(0, device=cuda)]) == 0


def test_refusals(cuda):
    a, b = torch.randn(8, device=cuda), torch.randn(8, 8, device=cuda)
    for bad in (lambda: hp.grad_norm([a.double()]), lambda: hp.grad_norm([a.cpu()]),
                lambda: hp.grad_norm([b.t()]), lambda: hp.clip_grad_norm([a], -1.0),
                lambda: hp.clip_grad_norm([a], float("nan")),
                lambda: hp.clip_grad_norm([a], 1.0, out=[a[:4]]),
                lambda: hp.clip_grad_norm([a], 1.0, out=[a, b]),
                lambda: hp.clip_grad_norm([b[0:4].view(-1)], 1.0, out=[b.view(-1)[1:33]])):
        with pytest.raises(RuntimeError):
            bad()


def test_strided_sums_are_short(cuda):
    """A chunk of a strided tensor is summed like one of a dense tensor: a thread's 256 terms in
    eight sums of 32.  The first term of each thread's is 1, the others half its last place, which
    vanish one by one beside it and count where they are summed among themselves."""
    n = 77_000_000  # enough for the longest chunks, 65536 elements
    flat = torch.full((n,), (0.98 * 2.0 ** -24) ** 0.5, device=cuda)
    flat[:n // 65536 * 65536].view(-1, 65536)[:, :256] = 1
    g = torch.zeros(n // 1000, 1024, device=cuda)[:, :1000]
    g.copy_(flat.view(-1, 1000))
    want = flat.double().square().sum().sqrt()
    # 32 terms, 3 joins of the eight sums, 5 in a warp and 7 of the warps, 2^-24 each;
    # half of that in the root, and its own rounding.
    bound = (47 / 2 + 1) * 2.0 ** -24 * want.item()
    assert abs(hp.grad_norm([flat]).item() - want.item()) <= bound
    assert abs(hp.grad_norm([g]).item() - want.item()) <= bound
