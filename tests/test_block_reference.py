"""The 64-bit formulas of the gated norms' and the log probabilities' gradients against central
differences of their definitions (CPU): what the kernels are compared with is itself checked."""
import pytest
import torch

from tests import block_reference as B

H = 1e-5
# Central differences are off by H^2 f''' / 6 (1e-10 here) and by 1e-16 f / H (1e-10 for f about
# 10): 1e-7 leaves both far behind.
CLOSE = dict(rtol=1e-6, atol=1e-7)


def differences(f, t):
    out = torch.empty_like(t)
    flat, o = t.view(-1), out.view(-1)
    for k in range(flat.numel()):
        v = flat[k].item()
        flat[k] = v + H
        hi = f()
        flat[k] = v - H
        lo = f()
        flat[k] = v
        o[k] = (hi - lo) / (2 * H)
    return out


def normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", [None, (5,), (2, 3, 1), (2, 1, 5), (2, 3, 5), (2, 1, 1), (1,)], ids=str)
def test_gated_norm(gate, post):
    x, r, d, e = (normal(2, 3, 5, seed=k) for k in range(4))
    p, w = (normal(5, seed=4) if post else None), normal(5, seed=5)
    g = None if gate is None else normal(*gate, seed=6)

    def f():
        (out, _), (total, _) = B.gated_add_rms_norm(x, r, p, w, 1e-6, g, 0.7)
        return float((out * d).sum() + (total * e).sum())

    total = B.gated_add_rms_norm(x, r, p, w, 1e-6, g, 0.7)[1][0]
    found = B.gated_add_rms_norm_backward(d, x, total, p, w, 1e-6, g, 0.7, e)
    leaves = {"x": x, "residual": r, "weight": w, "post_weight": p, "gate": g}
    assert set(found) == {k for k, v in leaves.items() if v is not None}
    for name, (value, bound) in found.items():
        assert (bound >= 0).all()
        torch.testing.assert_close(value, differences(f, leaves[name]), **CLOSE)


@pytest.mark.parametrize("entropy", [True, False])
def test_log_probs(entropy):
    x, w, c, h = normal(4, 5, seed=3), normal(7, 5, seed=4), normal(4, seed=5), normal(4, seed=6)
    t = torch.tensor([0, 6, -100, 3])

    def f():
        log_prob, ent, _, _ = B.log_probs(x, w, t, -100, 0.8)
        return float((log_prob * c).sum() + ((ent * h).sum() if entropy else 0))

    dx, dw, _, err = B.log_probs_backward(c, x, w, t, -100, 0.8, h if entropy else None)
    torch.testing.assert_close(dx, differences(f, x), **CLOSE)
    torch.testing.assert_close(dw, differences(f, w), **CLOSE)
    assert not dx[2].any() and (err >= 0).all()
