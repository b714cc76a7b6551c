"""The training operators as measured cases: a gated linear layer, the linear
cross entropy over a vocabulary, RMSNorm's backward pass and gradient clipping,
each with its plain form in 32 bits and its definition in 64 bits.

A case is a dict of plain values.  ``op`` names the operator:

gated  h = act(x Wg^T) * (x Wu^T), ``weight`` holding the rows [Wg; Wu]; with
       ``train`` also the gradients of x and weight for a given gradient of h.
loss   per-row cross entropy of softmax(x W^T) against target indices; rows
       whose target is -100 are left out; with ``train`` also the gradients of
       x and W for a given gradient of each row's loss.
norm   gradients of RMSNorm's input and weight, optionally with the gradient
       that reaches the same input through the residual branch added.
clip   the 2-norm of all gradients of a model and the clipped gradients,
       written to buffers of the optimiser's type.
"""
import math

import torch

own = False

IGNORE = -100
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One token of one sequence through a feed-forward block's first half: latency and weight bandwidth.
        {"name": "gated_token", "op": "gated", "rows": 1, "hidden": 4096, "d": 14336, "dtype": "bf16", "act": "silu", "pad": 0, "train": False},
        # A decode batch of a wide model; the rows are slices of a wider buffer.
        {"name": "gated_decode", "op": "gated", "rows": 48, "hidden": 8192, "d": 28672, "dtype": "fp16", "act": "gelu_tanh", "pad": 64, "train": False},
        # A training step's tokens of one device: forward and backward.
        {"name": "gated_train", "op": "gated", "rows": 4096, "hidden": 4096, "d": 14336, "dtype": "bf16", "act": "silu", "pad": 0, "train": True},
        # A ragged batch on sizes that are no multiple of anything: forward and backward.
        {"name": "gated_odd", "op": "gated", "rows": 517, "hidden": 1001, "d": 2731, "dtype": "fp16", "act": "gelu", "pad": 0, "train": True},
        # Scoring a few candidate tokens: the smallest call of the loss.
        {"name": "loss_few", "op": "loss", "rows": 7, "hidden": 1024, "vocab": 32768, "dtype": "bf16", "ignored": 0.0, "train": False},
        # Perplexity of a batch of documents: the loss alone, an odd vocabulary.
        {"name": "loss_eval", "op": "loss", "rows": 2048, "hidden": 5120, "vocab": 100003, "dtype": "fp16", "ignored": 0.1, "train": False},
        # A training step's tokens over a large vocabulary: the largest case.
        {"name": "loss_train", "op": "loss", "rows": 8192, "hidden": 4096, "vocab": 131072, "dtype": "bf16", "ignored": 0.05, "train": True},
        # Fine-tuning on the answers alone: most rows are left out, odd sizes.
        {"name": "loss_odd", "op": "loss", "rows": 1023, "hidden": 2056, "vocab": 50001, "dtype": "bf16", "ignored": 0.7, "train": True},
        # The norm of a training step with the residual branch's gradient.
        {"name": "norm_train", "op": "norm", "rows": 4096, "hidden": 8192, "dtype": "bf16", "residual": True},
        # A few rows of an odd width, without a residual.
        {"name": "norm_odd", "op": "norm", "rows": 33, "hidden": 5001, "dtype": "fp16", "residual": False},
        # A small model: latency over a few dozen tensors of odd sizes.
        {"name": "clip_small", "op": "clip", "layers": 4, "hidden": 255, "d": 701, "vocab": 1001, "dtype": "bf16", "out": "bf16"},
        # A larger one, 16-bit gradients into 32-bit buffers.
        {"name": "clip_large", "op": "clip", "layers": 24, "hidden": 2048, "d": 5632, "vocab": 32768, "dtype": "bf16", "out": "fp32"},
    ]


MOST = None


def draw(rng):
    global MOST
    if MOST is None:
        w = [work(c) for c in listed()]
        MOST = {k: max(x[k] for x in w) for k in ("flops", "bytes")}

    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return n if rng.random() < 0.3 else max(lo, n // 8 * 8)

    while True:
        op, dtype = rng.choice(("gated", "loss", "norm", "clip")), rng.choice(("bf16", "fp16"))
        if op == "gated":
            case = {"op": op, "rows": size(1, 8192), "hidden": size(256, 8192), "d": size(256, 28672), "dtype": dtype,
                    "act": rng.choice(("silu", "gelu", "gelu_tanh")), "pad": rng.choice((0, 0, 8, 64)), "train": rng.random() < 0.5}
        elif op == "loss":
            case = {"op": op, "rows": size(1, 8192), "hidden": size(256, 8192), "vocab": size(1000, 131072), "dtype": dtype,
                    "ignored": rng.choice((0.0, 0.1, 0.7)), "train": rng.random() < 0.5}
        elif op == "norm":
            case = {"op": op, "rows": size(1, 16384), "hidden": size(256, 32768), "dtype": dtype, "residual": rng.random() < 0.5}
        else:
            case = {"op": op, "layers": size(1, 32), "hidden": size(128, 2048), "d": size(256, 8192), "vocab": size(1000, 65536),
                    "dtype": rng.choice(("bf16", "fp16", "fp32")), "out": rng.choice(("same", "fp32"))}
            case["out"] = case["dtype"] if case["out"] == "same" else "fp32"
        w = work(case)
        if 1e5 < w["bytes"] <= MOST["bytes"] and w["flops"] <= MOST["flops"] / 2:
            return case


def shapes(case):
    """The parameters of a transformer, as its gradients come."""
    h, d = case["hidden"], case["d"]
    layer = [(h,), (3 * h, h), (h, h), (h,), (2 * d, h), (h, d)]
    return [(case["vocab"], h)] + layer * case["layers"] + [(h,)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)

    s = {"case": case}
    if case["op"] == "gated":
        m, h, d = case["rows"], case["hidden"], case["d"]
        s["x"] = normal(m, h + case["pad"])[:, :h]
        s["weight"] = normal(2 * d, h, scale=h ** -0.5)
        if case["train"]:
            s["grad_out"] = normal(m, d, scale=0.1)
    elif case["op"] == "loss":
        m, h, v = case["rows"], case["hidden"], case["vocab"]
        s["x"], s["weight"] = normal(m, h), normal(v, h, scale=2.0 * h ** -0.5)
        s["target"] = torch.randint(0, v, (m,), generator=g, device="cuda")
        s["target"][torch.rand(m, generator=g, device="cuda") < case["ignored"]] = IGNORE
        # The mean over the rows that count, times a loss scale that keeps 16-bit gradients in range.
        s["grad_loss"] = torch.full((m,), 256.0, device="cuda") / (s["target"] != IGNORE).sum().clamp(min=1)
    elif case["op"] == "norm":
        m, h = case["rows"], case["hidden"]
        s["x"], s["grad_out"] = normal(m, h), normal(m, h, scale=0.1)
        s["weight"] = (1.0 + 0.1 * torch.randn(h, generator=g, device="cuda")).to(t)
        s["grad_residual"] = normal(m, h, scale=0.1) if case["residual"] else None
    else:
        sizes = [math.prod(x) for x in shapes(case)]
        flat = normal(sum(sizes), scale=0.01)
        s["out"] = torch.empty(sum(sizes), dtype=TYPES[case["out"]], device="cuda")
        s["grads"] = [x.view(y) for x, y in zip(flat.split(sizes), shapes(case))]
        s["outs"] = [x.view(y) for x, y in zip(s["out"].split(sizes), shapes(case))]
        s["max_norm"] = 1.0
    return s


def run(s):
    case = s["case"]
    return (run_own if own else run_plain)[case["op"]](s, case)


def own_gated(s, case):
    import hp_rms_norm_b200 as hp

    if not case["train"]:
        return {"out": hp.gated_linear(s["x"], s["weight"], case["act"])}
    gate_up = torch.empty(case["rows"], 2 * case["d"], dtype=torch.float32, device="cuda")
    out = hp.gated_linear(s["x"], s["weight"], case["act"], gate_up=gate_up)
    dx, dw = hp.gated_linear_backward(s["grad_out"], s["x"], s["weight"], case["act"], gate_up=gate_up)
    return {"out": out, "grad_x": dx, "grad_weight": dw}


def own_loss(s, case):
    import hp_rms_norm_b200 as hp

    loss, lse = hp.linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=IGNORE)
    if not case["train"]:
        return {"loss": loss}
    dx, dw = hp.linear_cross_entropy_backward(s["grad_loss"], s["x"], s["weight"], s["target"], lse, ignore_index=IGNORE)
    return {"loss": loss, "grad_x": dx, "grad_weight": dw}


def own_norm(s, case):
    import hp_rms_norm_b200 as hp

    dx, dw = hp.rms_norm_backward(s["grad_out"], s["x"], s["weight"], EPS, grad_residual=s["grad_residual"])
    return {"grad_x": dx, "grad_weight": dw}


def own_clip(s, case):
    import hp_rms_norm_b200 as hp

    return {"norm": hp.clip_grad_norm(s["grads"], s["max_norm"], out=s["outs"]), "out": s["out"]}


def act_and_slope(a, act):
    """act(a) and its derivative."""
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-a))
        return a * q, q * (1.0 + a * (1.0 - q))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(a * 0.5 ** 0.5))
        return a * c, c + a * torch.exp(-0.5 * a * a) * (2.0 * math.pi) ** -0.5
    k = (2.0 / math.pi) ** 0.5
    q = torch.tanh(k * (a + 0.044715 * a * a * a))
    return 0.5 * a * (1.0 + q), 0.5 * (1.0 + q) + 0.5 * a * (1.0 - q * q) * k * (1.0 + 3.0 * 0.044715 * a * a)


def plain_gated(s, case):
    t, d = s["x"].dtype, case["d"]
    x, w = s["x"].float(), s["weight"].float()
    gate_up = x @ w.T
    gate, up = gate_up[:, :d], gate_up[:, d:]
    a, slope = act_and_slope(gate, case["act"])
    out = (a * up).to(t)
    if not case["train"]:
        return {"out": out}
    g = s["grad_out"].float()
    grad = torch.cat((g * up * slope, g * a), 1)
    return {"out": out, "grad_x": (grad @ w).to(t), "grad_weight": (grad.T @ x).to(t)}


def plain_loss(s, case):
    t, target = s["x"].dtype, s["target"]
    x, w = s["x"].float(), s["weight"].float()
    logits = x @ w.T
    top = logits.max(1, keepdim=True).values
    lse = top[:, 0] + torch.log(torch.exp(logits - top).sum(1))
    counts = target != IGNORE
    at = torch.where(counts, target, torch.zeros_like(target))[:, None]
    loss = torch.where(counts, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
    if not case["train"]:
        return {"loss": loss}
    grad = logits.sub_(lse[:, None]).exp_()
    grad.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
    grad.mul_((s["grad_loss"] * counts)[:, None])
    return {"loss": loss, "grad_x": (grad @ w).to(t), "grad_weight": (grad.T @ x).to(t)}


def plain_norm(s, case):
    t = s["x"].dtype
    x, w, g = s["x"].float(), s["weight"].float(), s["grad_out"].float()
    inv = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    n = x * inv
    wg = g * w
    dx = inv * (wg - n * (wg * n).mean(1, keepdim=True))
    if s["grad_residual"] is not None:
        dx = dx + s["grad_residual"].float()
    return {"grad_x": dx.to(t), "grad_weight": (g * n).sum(0).to(t)}


def plain_clip(s, case):
    norm = torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [y.copy_(x.float() * scale) for x, y in zip(s["grads"], s["outs"])]
    return {"norm": norm, "out": s["out"]}


run_own = {"gated": own_gated, "loss": own_loss, "norm": own_norm, "clip": own_clip}
run_plain = {"gated": plain_gated, "loss": plain_loss, "norm": plain_norm, "clip": plain_clip}


def work(case):
    e = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "gated":
        m, h, d = case["rows"], case["hidden"], case["d"]
        n = {"bytes": e * (m * h + 2 * d * h + m * d), "flops": 4 * m * h * d}
        if case["train"]:  # the gradients of x and weight for a gradient of the output, the products kept
            n = {"bytes": n["bytes"] + e * (m * d + m * h + 2 * d * h), "flops": n["flops"] + 8 * m * h * d}
    elif case["op"] == "loss":
        m, h, v = case["rows"], case["hidden"], case["vocab"]
        n = {"bytes": e * (m * h + v * h) + 12 * m, "flops": 2 * m * v * h}
        if case["train"]:
            n = {"bytes": n["bytes"] + e * (m * h + v * h) + 4 * m, "flops": n["flops"] + 4 * m * v * h}
    elif case["op"] == "norm":
        m, h = case["rows"], case["hidden"]
        n = {"bytes": e * (m * h * (4 if case["residual"] else 3) + 2 * h), "flops": 12 * m * h}
    else:
        k = sum(math.prod(x) for x in shapes(case))
        n = {"bytes": k * (e + (4 if case["out"] == "fp32" else 2)), "flops": 3 * k}
    return n


def exact(case, seed):
    """The definitions in 64 bits, gradients by automatic differentiation."""
    s = prepare(case, seed)
    if case["op"] == "clip":
        flat = torch.cat([x.reshape(-1) for x in s["grads"]]).double()
        norm = torch.linalg.vector_norm(flat)
        return {"norm": norm, "out": flat * min(1.0, s["max_norm"] / (norm.item() + 1e-6))}
    x, w = s["x"].double().requires_grad_(), s["weight"].double().requires_grad_()
    train = case.get("train", True)
    with torch.set_grad_enabled(train):
        if case["op"] == "gated":
            gate, up = torch.nn.functional.linear(x, w).chunk(2, dim=1)
            act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
                   "gelu_tanh": lambda a: torch.nn.functional.gelu(a, approximate="tanh")}[case["act"]]
            y, name = act(gate) * up, "out"
        elif case["op"] == "loss":
            logits = torch.nn.functional.linear(x, w)
            y, name = torch.nn.functional.cross_entropy(logits, s["target"], ignore_index=IGNORE, reduction="none"), "loss"
        else:
            y, name = x * (x.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5) * w, None
    found = {} if name is None else {name: y.detach()}
    if train:
        grad = s["grad_loss"] if case["op"] == "loss" else s["grad_out"]
        dx, dw = torch.autograd.grad(y, (x, w), grad.double())
        if s.get("grad_residual") is not None:
            dx = dx + s["grad_residual"].double()
        found |= {"grad_x": dx, "grad_weight": dw}
    return found
