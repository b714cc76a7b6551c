"""Run as a process of its own: the training operators' first calls are inside a CUDA graph
capture; prints OK when replays give what later eager calls give."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import hp_rms_norm_b200 as hp  # noqa: E402


def main():
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(200, 256, generator=g, device="cuda").bfloat16()
    w = (torch.randn(320, 256, generator=g, device="cuda") / 16).bfloat16()
    dout = torch.randn(200, 160, generator=g, device="cuda").bfloat16()
    odd = torch.randn(200, 129, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 320, (200,), generator=g, device="cuda")
    c = torch.ones(200, device="cuda")
    grads = [torch.randn(n, generator=g, device="cuda") for n in (5000, 33)]

    def step():
        loss, lse = hp.linear_cross_entropy(x, w, t)
        out = [torch.empty_like(v) for v in grads]
        return (hp.gated_linear(x, w), *hp.gated_linear_backward(dout, x, w), loss,
                *hp.linear_cross_entropy_backward(c, x, w, t, lse),
                *hp.rms_norm_backward(x, x, x[0].contiguous(), 1e-6),
                *hp.rms_norm_backward(odd, odd, odd[0].contiguous(), 1e-6),
                hp.clip_grad_norm(grads, 1.0, out=out), *out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    eager = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, eager))
    print("OK")


if __name__ == "__main__":
    main()
