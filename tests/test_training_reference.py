"""The 64-bit formulas of the training operators' gradients against central differences of the
operators' definitions (CPU): what the kernels are compared with is itself checked."""
import pytest
import torch

from tests import training_reference as R

H = 1e-5


def differences(f, t):
    """Central differences of the scalar f() in every element of t (changed in place)."""
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


# Central differences are off by H^2 f''' / 6 (1e-10 here) and by 1e-16 f / H
# (1e-10 for f about 10): 1e-7 leaves both far behind.
CLOSE = dict(rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_linear(act):
    x, w, d = normal(3, 5, seed=0), normal(8, 5, seed=1), normal(3, 4, seed=2)
    f = lambda: float((R.gated_linear(x, w, act)[0] * d).sum())
    dx, dw, _ = R.gated_linear_backward(d, x, w, act)
    torch.testing.assert_close(dx, differences(f, x), **CLOSE)
    torch.testing.assert_close(dw, differences(f, w), **CLOSE)


def test_linear_cross_entropy():
    x, w, c = normal(4, 5, seed=3), normal(7, 5, seed=4), normal(4, seed=5)
    t = torch.tensor([0, 6, -100, 3])
    f = lambda: float((R.linear_cross_entropy(x, w, t, -100)[0] * c).sum())
    dx, dw, _ = R.linear_cross_entropy_backward(c, x, w, t, -100)
    torch.testing.assert_close(dx, differences(f, x), **CLOSE)
    torch.testing.assert_close(dw, differences(f, w), **CLOSE)
    assert not dx[2].any()


def test_rms_norm():
    x, w, d = normal(3, 6, seed=6), normal(6, seed=7), normal(3, 6, seed=8)
    f = lambda: float((x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w * d).sum())
    dx, dw = R.rms_norm_backward(d, x, w, 1e-6)
    torch.testing.assert_close(dx, differences(f, x), **CLOSE)
    torch.testing.assert_close(dw, differences(f, w), **CLOSE)
