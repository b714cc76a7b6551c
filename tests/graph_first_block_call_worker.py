"""Run as a process of its own: the first calls of the operators around a block are inside a CUDA
graph capture; prints OK when replays give what later eager calls give."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import hp_rms_norm_b200 as hp  # noqa: E402


def main():
    g = torch.Generator(device="cuda").manual_seed(0)
    x, r = (torch.randn(200, 256, generator=g, device="cuda").bfloat16() for _ in range(2))
    odd = torch.randn(200, 129, generator=g, device="cuda").bfloat16()
    w = (torch.randn(320, 256, generator=g, device="cuda") / 16).bfloat16()
    w8 = torch.randint(-127, 128, (320, 256), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(320, generator=g, device="cuda")
    p = torch.ones(256, device="cuda").bfloat16()
    t = torch.randint(0, 320, (200,), generator=g, device="cuda")
    c = torch.ones(200, device="cuda")

    def step():
        total = torch.empty_like(r)
        out = hp.gated_add_rms_norm(x, r, p, p, 1e-6, gate=p, residual_out=total)
        q, s = hp.rms_norm_int8(x, p, 1e-6)
        f = hp.linear_log_probs(x, w, t, top=4)
        few = hp.linear_log_probs(x[:5], w, t[:5], top=4)
        return (out, total, *hp.gated_add_rms_norm_backward(x, x, total, p, p, 1e-6, gate=p),
                *hp.gated_add_rms_norm_backward(odd, odd, odd, odd[0].clone(), odd[1].clone(), 1e-6)[:4],
                q, s, hp.linear_int8(q, s, w8, ws), hp.linear_int8(q[:3], s[:3], w8, ws), *f, *few,
                *hp.linear_log_probs_backward(c, x, w, t, f.lse, f.entropy, c))

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
