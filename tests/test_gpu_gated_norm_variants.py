"""The gated norm's backward pass against the 64-bit formulas where its kernels differ: gates that few
rows share, every kind of gate at every number of words a thread has, rows that start anywhere, rows
too long for the ring of rows in shared memory."""
import pytest
import torch

import hp_rms_norm_b200 as hp
from tests.test_gpu_gated_norm import EPS, check, make

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
