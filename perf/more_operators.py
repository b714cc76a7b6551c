"""More operators as measured cases: the norms on both sides of a gated block,
the log probabilities of given tokens with their entropy and best alternatives,
and the products of 8-bit integers with the norm that feeds them.  Each has its
plain form in 32 bits and its definition in 64 bits.

A case is a dict of plain values.  ``op`` names the operator:

block  residual' = scale * residual + gate * RMSNorm(x) * post_weight and
       out = RMSNorm(residual') * weight; ``gate`` is 'none', 'channel' (one
       value for each of the hidden channels), 'token' (one for each row),
       'sequence' (each sequence its own channels) or 'full' (one for each
       element); with ``train`` also the gradients of all five inputs.
logp   for L = x W^T / temperature the log probability of each row's target,
       the entropy of softmax(L) and the ``top`` largest log probabilities with
       their indices; rows whose target is -100 have neither log probability
       nor entropy (both 0).  With ``train`` also the gradients of x and W.
int8   out = (codes_x codes_w^T) scale_x scale_w + bias: 8-bit integers with a
       scale for each token and each output channel.
norm8  residual' = residual + x, RMSNorm(residual') * weight rounded to 8-bit
       integers with a scale for each token, and the int8 product of those.
"""
import math

import torch

own = False

IGNORE = -100
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One token of one sequence between two blocks: latency.
        {"name": "block_token", "op": "block", "rows": 1, "hidden": 4096, "dtype": "bf16", "gate": "channel", "sequences": 1, "post": True, "scale": 1.0, "train": False},
        # A training step's tokens of one device, forward and backward.
        {"name": "block_train", "op": "block", "rows": 4096, "hidden": 8192, "dtype": "bf16", "gate": "channel", "sequences": 1, "post": True, "scale": 1.0, "train": True},
        # Gates made for each sequence from its conditioning, odd sizes, a scaled residual.
        {"name": "block_sequences", "op": "block", "rows": 12 * 257, "hidden": 1001, "dtype": "fp16", "gate": "sequence", "sequences": 12, "post": True, "scale": 0.75, "train": True},
        # The next token of a few requests with five alternatives each: latency.
        {"name": "logp_few", "op": "logp", "rows": 7, "hidden": 1024, "vocab": 32768, "dtype": "bf16", "top": 5, "temperature": 1.0, "ignored": 0.0, "train": False},
        # Scoring a batch of documents over an odd vocabulary.
        {"name": "logp_score", "op": "logp", "rows": 2048, "hidden": 5120, "vocab": 100003, "dtype": "fp16", "top": 0, "temperature": 1.0, "ignored": 0.1, "train": False},
        # A prompt's tokens with twenty alternatives each.
        {"name": "logp_alternatives", "op": "logp", "rows": 512, "hidden": 4096, "vocab": 131072, "dtype": "bf16", "top": 20, "temperature": 1.0, "ignored": 0.0, "train": False},
        # A step of policy-gradient training with an entropy term, the tokens sampled at 0.8: the largest case.
        {"name": "logp_train", "op": "logp", "rows": 4096, "hidden": 4096, "vocab": 131072, "dtype": "bf16", "top": 0, "temperature": 0.8, "ignored": 0.3, "train": True},
        # A decode batch through a feed-forward block's first products: weight bandwidth.
        {"name": "int8_decode", "op": "int8", "rows": 16, "hidden": 4096, "out": 28672, "dtype": "bf16", "bias": False},
        # Prompts through a wide layer.
        {"name": "int8_prompt", "op": "int8", "rows": 8192, "hidden": 8192, "out": 28672, "dtype": "bf16", "bias": False},
        # A ragged batch on sizes that are no multiple of anything, with a bias.
        {"name": "int8_odd", "op": "int8", "rows": 517, "hidden": 2731, "out": 1001, "dtype": "fp16", "bias": True},
        # One token through a norm and the products after it.
        {"name": "norm8_token", "op": "norm8", "rows": 1, "hidden": 4096, "out": 6144, "dtype": "bf16"},
        # A prompt through a norm and the products after it.
        {"name": "norm8_prompt", "op": "norm8", "rows": 4096, "hidden": 8192, "out": 10240, "dtype": "bf16"},
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
        op, dtype = rng.choice(("block", "logp", "int8", "norm8")), rng.choice(("bf16", "fp16"))
        if op == "block":
            case = {"op": op, "rows": size(1, 8192), "hidden": size(64, 16384), "dtype": dtype,
                    "gate": rng.choice(("none", "channel", "token", "sequence", "full")), "sequences": 1,
                    "post": rng.random() < 0.8, "scale": rng.choice((1.0, 0.5)), "train": rng.random() < 0.6}
            if case["gate"] == "sequence":
                case["sequences"] = rng.randint(1, 32)
                case["rows"] = case["sequences"] * max(1, case["rows"] // case["sequences"])
        elif op == "logp":
            train = rng.random() < 0.4
            case = {"op": op, "rows": size(1, 8192), "hidden": size(256, 8192), "vocab": size(1000, 131072), "dtype": dtype,
                    "top": 0 if train else rng.choice((0, 1, 5, 20)), "temperature": rng.choice((1.0, 0.8)),
                    "ignored": rng.choice((0.0, 0.1, 0.5)), "train": train}
        elif op == "int8":
            case = {"op": op, "rows": size(1, 8192), "hidden": size(256, 28672), "out": size(256, 28672), "dtype": dtype,
                    "bias": rng.random() < 0.3}
        else:
            case = {"op": op, "rows": size(1, 8192), "hidden": size(256, 16384), "out": size(256, 16384), "dtype": dtype}
        w = work(case)
        if 1e5 < w["bytes"] <= MOST["bytes"] and w["flops"] <= MOST["flops"] / 2:
            return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).add_(mean).to(dtype)

    s = {"case": case}
    m, h = case["rows"], case["hidden"]
    if case["op"] == "block":
        shape = (case["sequences"], m // case["sequences"], h) if case["gate"] == "sequence" else (m, h)
        s["x"], s["residual"] = normal(*shape), normal(*shape, scale=3.0)
        s["post_weight"] = normal(h, scale=0.1, mean=0.5) if case["post"] else None
        s["weight"] = normal(h, scale=0.1, mean=1.0)
        gates = {"none": None, "channel": (h,), "token": (m, 1), "sequence": (case["sequences"], 1, h), "full": (m, h)}
        s["gate"] = None if case["gate"] == "none" else normal(*gates[case["gate"]], scale=0.2, mean=0.8)
        s["residual_out"], s["out"] = torch.empty_like(s["residual"]), torch.empty_like(s["x"])
        if case["train"]:
            s["grad_out"], s["grad_residual"] = normal(*shape, scale=0.1), normal(*shape, scale=0.1)
    elif case["op"] == "logp":
        v = case["vocab"]
        s["x"], s["weight"] = normal(m, h), normal(v, h, scale=2.0 * h ** -0.5)
        s["target"] = torch.randint(0, v, (m,), generator=g, device="cuda")
        # The first row always counts.
        s["target"][1:][torch.rand(m, generator=g, device="cuda")[1:] < case["ignored"]] = IGNORE
        if case["train"]:
            # Advantages, and the weight of the entropy, over the rows that count, times a loss scale.
            n = 256.0 / (s["target"] != IGNORE).sum().clamp(min=1)
            s["grad_log_prob"] = normal(m, dtype=torch.float32) * n
            s["grad_entropy"] = torch.full((m,), 0.01, device="cuda") * n
    else:
        n = case["out"]
        w = normal(n, h, scale=h ** -0.5, dtype=torch.float32)
        s["weight_scale"] = w.abs().amax(1) / 127
        s["weight8"] = torch.round(w / s["weight_scale"][:, None]).to(torch.int8)
        if case["op"] == "int8":
            x = normal(m, h, dtype=torch.float32)
            s["x_scale"] = x.abs().amax(1) / 127
            s["x8"] = torch.round(x / s["x_scale"][:, None]).to(torch.int8)
            s["bias"] = normal(n) if case["bias"] else None
        else:
            s["x"], s["residual"], s["weight"] = normal(m, h), normal(m, h, scale=3.0), normal(h, scale=0.1, mean=1.0)
            s["residual_out"] = torch.empty_like(s["residual"])
        s["type"] = t
    return s


def run(s):
    case = s["case"]
    return (run_own if own else run_plain)[case["op"]](s, case)


def own_block(s, case):
    import hp_rms_norm_b200 as hp

    out = hp.gated_add_rms_norm(s["x"], s["residual"], s["post_weight"], s["weight"], EPS, gate=s["gate"],
                                residual_scale=case["scale"], out=s["out"], residual_out=s["residual_out"])
    found = {"out": out, "residual": s["residual_out"]}
    if not case["train"]:
        return found
    dx, dr, dp, dw, dg = hp.gated_add_rms_norm_backward(
        s["grad_out"], s["x"], s["residual_out"], s["post_weight"], s["weight"], EPS, gate=s["gate"],
        residual_scale=case["scale"], grad_residual=s["grad_residual"])
    return found | named_gradients(dx, dr, dp, dw, dg)


def named_gradients(dx, dr, dp, dw, dg):
    found = {"grad_x": dx, "grad_residual": dr, "grad_post_weight": dp, "grad_weight": dw, "grad_gate": dg}
    return {k: v for k, v in found.items() if v is not None}


def own_logp(s, case):
    import hp_rms_norm_b200 as hp

    log_prob, entropy, lse, top, at = hp.linear_log_probs(s["x"], s["weight"], s["target"], top=case["top"],
                                                          temperature=case["temperature"], ignore_index=IGNORE)
    found = {"log_prob": log_prob, "entropy": entropy}
    if case["top"]:
        found |= {"top_log_probs": top, "top_indices": at}
    if case["train"]:
        dx, dw = hp.linear_log_probs_backward(s["grad_log_prob"], s["x"], s["weight"], s["target"], lse, entropy=entropy,
                                              grad_entropy=s["grad_entropy"], temperature=case["temperature"],
                                              ignore_index=IGNORE)
        found |= {"grad_x": dx, "grad_weight": dw}
    return found


def own_int8(s, case):
    import hp_rms_norm_b200 as hp

    return {"out": hp.linear_int8(s["x8"], s["x_scale"], s["weight8"], s["weight_scale"], bias=s["bias"], dtype=s["type"])}


def own_norm8(s, case):
    import hp_rms_norm_b200 as hp

    codes, scale = hp.rms_norm_int8(s["x"], s["weight"], EPS, residual=s["residual"], residual_out=s["residual_out"])
    return {"out": hp.linear_int8(codes, scale, s["weight8"], s["weight_scale"], dtype=s["type"]), "residual": s["residual_out"]}


def norm_parts(x):
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return inv, x * inv


def norm_grad(grad, inv, n):
    """The gradient of x for a gradient of n = x inv."""
    return inv * (grad - n * (grad * n).mean(-1, keepdim=True))


def plain_block(s, case):
    t = s["x"].dtype
    x, r, w = s["x"].float(), s["residual"].float(), s["weight"].float()
    gate = None if s["gate"] is None else s["gate"].float()
    post = None if s["post_weight"] is None else s["post_weight"].float()
    if post is None:
        y = x
    else:
        inv_x, n_x = norm_parts(x)
        y = n_x * post
    total = case["scale"] * r + (y if gate is None else gate * y)
    inv, n = norm_parts(total)
    found = {"out": (n * w).to(t), "residual": total.to(t)}
    if not case["train"]:
        return found
    g = s["grad_out"].float()
    lead = tuple(range(g.dim() - 1))
    to_total = norm_grad(g * w, inv, n) + s["grad_residual"].float()
    to_y = to_total if gate is None else to_total * gate
    to_gate = to_post = None
    if gate is not None:
        to_gate = to_total * y
        # The sum over what the gate was broadcast over.
        shape = (1,) * (g.dim() - gate.dim()) + tuple(gate.shape)
        over = [k for k in range(g.dim()) if shape[k] == 1 and g.shape[k] != 1]
        to_gate = (to_gate.sum(over, keepdim=True) if over else to_gate).reshape(gate.shape).to(t)
    if post is None:
        to_x = to_y
    else:
        to_post = (to_y * n_x).sum(lead).to(t)
        to_x = norm_grad(to_y * post, inv_x, n_x)
    return found | named_gradients(to_x.to(t), (case["scale"] * to_total).to(t), to_post, (g * n).sum(lead).to(t), to_gate)


def plain_logp(s, case):
    t, target = s["x"].dtype, s["target"]
    x, w = s["x"].float(), s["weight"].float()
    inv_t = 1.0 / case["temperature"]
    logits = (x @ w.T).mul_(inv_t)
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1)
    lse = top[:, 0] + torch.log(total)
    counts = target != IGNORE
    at = torch.where(counts, target, torch.zeros_like(target))[:, None]
    zero = torch.zeros_like(lse)
    log_prob = torch.where(counts, (logits.gather(1, at)[:, 0] - top[:, 0]) - torch.log(total), zero)
    entropy = torch.log(total) - (e * (logits - top)).sum(1) / total
    found = {"log_prob": log_prob, "entropy": torch.where(counts, entropy, zero)}
    del e
    if case["top"]:
        # Alternatives that differ in their last bits are told apart in 64 bits, equal ones by their indices.
        near = torch.topk(logits, min(case["top"] + 8, case["vocab"]), dim=1).indices.sort(1).values
        chosen = []
        for rows, ids in zip(s["x"].split(64), near.split(64)):
            exact_logits = (s["weight"][ids].double() @ rows.double()[:, :, None])[:, :, 0] / case["temperature"]
            value, order = exact_logits.sort(dim=1, descending=True, stable=True)
            chosen.append((value[:, :case["top"]], ids.gather(1, order)[:, :case["top"]]))
        value, ids = torch.cat([c[0] for c in chosen]), torch.cat([c[1] for c in chosen])
        found |= {"top_log_probs": (value - lse.double()[:, None]).float(), "top_indices": ids}
    if case["train"]:
        log_p = logits.sub_(lse[:, None])
        grad = -torch.exp(log_p)
        d = (s["grad_entropy"] * counts)[:, None]
        c = (s["grad_log_prob"] * counts)[:, None]
        grad.mul_((log_p + entropy[:, None]).mul_(d).add_(c))
        grad.scatter_add_(1, at, c)
        grad.mul_(inv_t)
        found |= {"grad_x": (grad @ w).to(t), "grad_weight": (grad.T @ x).to(t)}
    return found


def scaled_product(x8, x_scale, w8, w_scale, bias, t):
    # Sums of 28672 such products stay far below 2^24 here, so fp32 holds them exactly.
    y = (x8.float() @ w8.float().T) * x_scale[:, None] * w_scale
    return (y if bias is None else y + bias.float()).to(t)


def plain_int8(s, case):
    return {"out": scaled_product(s["x8"], s["x_scale"], s["weight8"], s["weight_scale"], s["bias"], s["type"])}


def plain_norm8(s, case):
    total = s["x"].float() + s["residual"].float()
    y = norm_parts(total)[1] * s["weight"].float()
    scale = y.abs().amax(1) / 127
    codes = torch.round(y / torch.where(scale > 0, scale, 1.0)[:, None])
    return {"out": scaled_product(codes, scale, s["weight8"], s["weight_scale"], None, s["type"]),
            "residual": total.to(s["type"])}


run_own = {"block": own_block, "logp": own_logp, "int8": own_int8, "norm8": own_norm8}
run_plain = {"block": plain_block, "logp": plain_logp, "int8": plain_int8, "norm8": plain_norm8}


def work(case):
    m, h = case["rows"], case["hidden"]
    if case["op"] == "block":
        gate = {"none": 0, "channel": h, "token": m, "sequence": case["sequences"] * h, "full": m * h}[case["gate"]]
        once = gate + (2 if case["post"] else 1) * h
        n = {"bytes": 2 * (4 * m * h + once), "flops": 12 * m * h}
        if case["train"]:  # two more gradients in, two out, and those of the weights and the gate
            n = {"bytes": n["bytes"] + 2 * (4 * m * h + once), "flops": 42 * m * h}
    elif case["op"] == "logp":
        v = case["vocab"]
        n = {"bytes": 2 * (m * h + v * h) + (16 + 12 * case["top"]) * m, "flops": 2 * m * v * h}
        if case["train"]:
            n = {"bytes": n["bytes"] + 2 * (m * h + v * h) + 8 * m, "flops": n["flops"] + 4 * m * v * h}
    else:
        k = case["out"]
        n = {"bytes": k * h + 4 * k + 2 * m * k, "flops": 2 * m * k * h}
        if case["op"] == "int8":
            n["bytes"] += m * h + 4 * m + (2 * k if case["bias"] else 0)
        else:
            n["bytes"] += 6 * m * h + 2 * h
    return n


def exact(case, seed):
    """The definitions in 64 bits, gradients by automatic differentiation."""
    s = prepare(case, seed)
    if case["op"] == "block":
        leaves = {k: None if s[k] is None else s[k].double().requires_grad_()
                  for k in ("x", "residual", "post_weight", "weight", "gate")}

        def norm(a, weight):
            return a * (a.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5) * weight

        with torch.set_grad_enabled(case["train"]):
            y = leaves["x"] if leaves["post_weight"] is None else norm(leaves["x"], leaves["post_weight"])
            total = leaves["residual"] * case["scale"] + (y if leaves["gate"] is None else y * leaves["gate"])
            out = norm(total, leaves["weight"])
        found = {"out": out.detach(), "residual": total.detach()}
        if case["train"]:
            there = {k: v for k, v in leaves.items() if v is not None}
            grads = torch.autograd.grad((out, total), list(there.values()), (s["grad_out"].double(), s["grad_residual"].double()))
            found |= {"grad_" + k: v for k, v in zip(there, grads)}
        return found
    if case["op"] == "logp":
        x, w = s["x"].double().requires_grad_(case["train"]), s["weight"].double().requires_grad_(case["train"])
        counts = s["target"] != IGNORE
        with torch.set_grad_enabled(case["train"]):
            log_p = torch.log_softmax(torch.nn.functional.linear(x, w) / case["temperature"], -1)
            log_prob = log_p.gather(1, s["target"].clamp(min=0)[:, None])[:, 0] * counts
            entropy = -(log_p.exp() * log_p).sum(-1) * counts
        found = {"log_prob": log_prob.detach(), "entropy": entropy.detach()}
        if case["top"]:
            value, order = [], []
            for part in log_p.split(256):
                v, o = part.sort(dim=-1, descending=True, stable=True)
                value.append(v[:, :case["top"]].clone()), order.append(o[:, :case["top"]].clone())
            found |= {"top_log_probs": torch.cat(value), "top_indices": torch.cat(order)}
        if case["train"]:
            dx, dw = torch.autograd.grad((log_prob, entropy), (x, w), (s["grad_log_prob"].double(), s["grad_entropy"].double()))
            found |= {"grad_x": dx, "grad_weight": dw}
        return found
    weight = s["weight8"].double()
    if case["op"] == "int8":
        out = torch.nn.functional.linear(s["x8"].double() * s["x_scale"].double()[:, None], weight * s["weight_scale"].double()[:, None])
        return {"out": out if s["bias"] is None else out + s["bias"].double()}
    total = s["residual"].double() + s["x"].double()
    y = total * (total.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5) * s["weight"].double()
    step = y.abs().amax(-1, keepdim=True) / 127
    values = torch.round(y / step) * step
    return {"out": torch.nn.functional.linear(values, weight * s["weight_scale"].double()[:, None]), "residual": total}
