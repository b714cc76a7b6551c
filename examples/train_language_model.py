"""A training step of a small language model on the package's training operators.

    python examples/train_language_model.py [--steps 20] [--layers 4] [--hidden 512] ...

Each layer mixes the tokens before it (a plain causal mean, the place of an
attention layer) and runs a pre-norm gated feed-forward block; the loss is taken
over the vocabulary without its logits; all gradients are clipped together into
float32 buffers and applied to float32 master weights.  Synthetic data: a fixed
random permutation of the vocabulary has to be learnt.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import hp_rms_norm_b200 as hp  # noqa: E402
from hp_rms_norm_b200 import autograd as A  # noqa: E402


def parameters(layers, hidden, ffn, vocab, device, dtype):
    g = torch.Generator(device=device).manual_seed(0)

    def normal(*shape, scale):
        t = torch.randn(*shape, generator=g, device=device) * scale
        return t.to(dtype).requires_grad_()

    p = {"embedding": normal(vocab, hidden, scale=1.0), "head": normal(vocab, hidden, scale=hidden ** -0.5),
         "norm": torch.ones(hidden, device=device, dtype=dtype).requires_grad_()}
    for k in range(layers):
        p[f"{k}.norm"] = torch.ones(hidden, device=device, dtype=dtype).requires_grad_()
        p[f"{k}.gate_up"] = normal(2 * ffn, hidden, scale=hidden ** -0.5)
        p[f"{k}.down"] = normal(hidden, ffn, scale=(ffn * layers) ** -0.5)
    return p


def loss_of(p, layers, tokens, targets, eps=1e-6):
    residual = torch.nn.functional.embedding(tokens, p["embedding"])
    count = torch.arange(1, tokens.shape[1] + 1, device=tokens.device)[:, None]
    x = torch.zeros_like(residual)
    for k in range(layers):
        y, residual = A.fused_add_rms_norm(x, residual, p[f"{k}.norm"], eps)
        y = 0.9 * y + 0.1 * (y.float().cumsum(1) / count).to(y.dtype)
        x = torch.nn.functional.linear(A.gated_linear(y, p[f"{k}.gate_up"]), p[f"{k}.down"])
    y, _ = A.fused_add_rms_norm(x, residual, p["norm"], eps)
    return A.linear_cross_entropy(y, p["head"], targets)


def train(steps=20, layers=4, hidden=512, ffn=1408, vocab=4096, batch=8, length=256, lr=0.3, max_norm=1.0,
          dtype=torch.bfloat16, device="cuda"):
    """Runs `steps` steps; returns the losses, a float32 tensor on the device."""
    p = parameters(layers, hidden, ffn, vocab, device, dtype)
    names = list(p)
    master = [p[n].detach().float() for n in names]
    clipped = [torch.empty_like(m) for m in master]
    g = torch.Generator(device=device).manual_seed(1)
    successor = torch.randperm(vocab, generator=g, device=device)
    losses = torch.empty(steps, device=device)
    for step in range(steps):
        tokens = torch.randint(0, vocab, (batch, length), generator=g, device=device)
        loss = loss_of(p, layers, tokens, successor[tokens])
        grads = torch.autograd.grad(loss, [p[n] for n in names])
        hp.clip_grad_norm(grads, max_norm, out=clipped)
        with torch.no_grad():
            for n, m, c in zip(names, master, clipped):
                m.sub_(c, alpha=lr)
                p[n].copy_(m)
        losses[step] = loss.detach()
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("steps", 20), ("layers", 4), ("hidden", 512), ("ffn", 1408), ("vocab", 4096),
                        ("batch", 8), ("length", 256)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--lr", type=float, default=0.3)
    a = ap.parse_args()
    losses = train(**vars(a)).tolist()
    for step, loss in enumerate(losses):
        print(f"step {step:4d}  loss {loss:.4f}")


if __name__ == "__main__":
    main()
