"""What the differentiable forms keep for a backward pass, on CPU with the kernels replaced."""
import pytest
import torch

from hp_rms_norm_b200 import autograd as A


@pytest.fixture
def kept(monkeypatch):
    """The gate_up argument of each forward call."""
    seen = []

    def forward(input, weight, act, gate_up=None):
        seen.append(gate_up)
        return input.new_zeros(input.shape[:-1] + (weight.shape[0] // 2,))

    monkeypatch.setattr(A.ops, "gated_linear", forward)
    return seen


def tensors(needs_grad):
    return torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16, requires_grad=needs_grad)


def test_products_are_kept_for_a_backward_pass(kept):
    A.gated_linear(*tensors(True))
    assert kept[0].shape == (5, 6) and kept[0].dtype == torch.float32
    A.gated_linear(*tensors(True), keep_products=False)
    assert kept[1] is None


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_kept_without_a_graph(kept, mode):
    """An evaluation of a model in training: its weights ask for gradients, the call does not."""
    with mode():
        A.gated_linear(*tensors(True))
    A.gated_linear(*tensors(False))
    assert kept == [None, None]
