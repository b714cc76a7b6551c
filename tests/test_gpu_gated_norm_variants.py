"""The gated norm's backward pass against the 64-bit formulas where its kernels differ: gates that few
rows share, every kind of gate at every number of words a thread has, rows that start anywhere, rows
too long for the ring of rows in shared memory."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from hp_rms_norm_b200 import capi
from tests.test_gpu_gated_norm import EPS, GATES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("post", [True, False], ids=["post", "no post"])
@pytest.mark.parametrize("lead,hidden", [((2500, 2), 64), ((3, 2), 64), ((75, 2), 72), ((1036, 2), 64), ((700, 3), 128), ((149, 7), 128),
                                         ((5, 64), 200), ((900, 2), 203), ((50, 3), 1001), ((3, 1000), 61), ((400, 2), 1024),
                                         ((160, 5), 4096), ((37, 4), 12288)], ids=str)
def test_gates_that_few_rows_share(cuda, lead, hidden, post):
    """Fewer rows than groups of threads, runs that end inside a gate's rows, runs of one row, gates of
    more rows than a run."""
    check(make(lead, hidden, torch.float16, cuda, gate="sequence", post=post), 0.75, f"{lead} x {hidden}")


def test_the_same_bits_every_time(cuda):
    s = make((2500, 2), 64, torch.bfloat16, cuda, gate="sequence")
    calls = [hp.gated_add_rms_norm_backward(s["d"], s["x"], s["r"], s["p"], s["w"], EPS, gate=s["gate"], grad_residual=s["e"]) for _ in range(4)]
    for grads in calls[1:]:
        assert all(torch.equal(a, b) for a, b in zip(calls[0], grads))


# Words a thread: 8 to 7680 elements, 12 to 8448, 24 to 16896 (rows on 16-byte boundaries alone, and with
# a gate for every element to 14080); past that, and with rows off the boundaries from 8449, the kernels
# that read rows twice.
WIDE = [7688, 8192, 8448, 8456, 10240, 12288, 14080, 14088, 16384, 16896, 16904]
ODD = [7679, 7683, 8191, 8447, 8449, 10001, 16383, 33001]


@pytest.mark.parametrize("post", [True, False], ids=["post", "no post"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("hidden", WIDE)
def test_wide_rows(cuda, hidden, gate, post):
    check(make((3, 5), hidden, torch.bfloat16, cuda, gate=gate, post=post), 1.0, f"{hidden} {gate}")
    check(make((2, 4), hidden, torch.float16, cuda, gate=gate, post=post), 0.5, f"{hidden} {gate}", with_e=False)


@pytest.mark.parametrize("post", [True, False], ids=["post", "no post"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("hidden", ODD)
def test_wide_rows_that_start_anywhere(cuda, hidden, gate, post):
    check(make((3, 5), hidden, torch.float16, cuda, gate=gate, post=post), 1.0, f"{hidden} {gate}")
    check(make((2, 4), hidden, torch.bfloat16, cuda, gate=gate, post=post), 0.5, f"{hidden} {gate}", with_e=False)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("hidden", [8192, 12288, 16384])
def test_wide_rows_one_element_behind_a_boundary(cuda, hidden, gate):
    """Whole vectors, every tensor one element off; rows with gaps between them."""
    s = make((2, 3), hidden, torch.bfloat16, cuda, gate=gate)
    for k, v in s.items():
        if v is None or v.shape[-1] == 1:
            continue
        rows, gap = v.numel() // hidden, 0 if v.dim() == 1 else 5
        held = torch.full((1 + rows * (hidden + gap),), float("nan"), dtype=v.dtype, device=cuda)
        strides = [hidden + gap]
        for n in reversed(v.shape[1:-1]):
            strides.insert(0, strides[0] * n)
        at = held.as_strided(v.shape, (strides if v.dim() > 1 else []) + [1], 1)
        at.copy_(v)
        s[k] = at
    check(s, 0.75, f"{hidden} {gate}")


@pytest.mark.parametrize("gate", GATES)
def test_more_wide_rows_than_CTAs(cuda, gate):
    """Rings of one row that go round, sums over many runs."""
    check(make((2, 230), 12288, torch.bfloat16, cuda, gate=gate), 1.0, f"460 x 12288 {gate}")
    check(make((5, 64), 8200, torch.float16, cuda, gate=gate), 1.0, f"320 x 8200 {gate}")
    check(make((4, 41), 9001, torch.float16, cuda, gate=gate), 1.0, f"164 x 9001 {gate}")


def test_a_wait_that_runs_out_in_a_run_of_its_own(cuda):
    """The hook leaves out all loads: the launch ends, the count tells, later calls are refused until it
    is reset, and nothing is left behind."""
    s = make((2500, 2), 512, torch.bfloat16, cuda, gate="sequence")

    def call():
        return hp.gated_add_rms_norm_backward(s["d"], s["x"], s["r"], s["p"], s["w"], EPS, gate=s["gate"], grad_residual=s["e"])

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
    with pytest.raises(RuntimeError, match="ran out"):
        call()
    assert capi.wait_timeouts(reset=True) > 0
    got = call()
    torch.cuda.synchronize()
    assert capi.wait_timeouts() == 0 and all(torch.equal(a, b) for a, b in zip(want, got))
