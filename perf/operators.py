"""The operators of the training and evaluation of the text model around the latent code, in plain form and as the
framework's kernels, on cases of the sizes that they run at.

Operators: the cross entropy of a decoder's hidden states over the whole vocabulary with its gradients ("train"), the
log-likelihood of whole sequences for the importance-weighted estimate ("seq"), that of single tokens ("token"), and
the norm of all gradients together with their clipping ("clip").
"""
import math
import random

import torch

own = False

IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one training step's reconstruction term at the usual batch: 32 padded sentences of 64 tokens, a masked
        # language model's vocabulary and width, mixed precision
        {"name": "train bf16 32x64", "op": "train", "dtype": "bf16", "B": 32, "K": 1, "L": 64, "H": 768, "V": 50265,
         "bias": True, "pad": True, "banned": 0, "cut": True},
        # the same step in the type that the estimators have trained in so far
        {"name": "train f32 16x64", "op": "train", "dtype": "f32", "B": 16, "K": 1, "L": 64, "H": 768, "V": 50265,
         "bias": True, "pad": True, "banned": 0, "cut": True},
        # a large batch of full sequences and a wider model: the throughput end
        {"name": "train bf16 32x512", "op": "train", "dtype": "bf16", "B": 32, "K": 1, "L": 512, "H": 1024, "V": 50265,
         "bias": True, "pad": False, "banned": 0, "cut": False},
        # a small word-level model: odd sizes throughout, no bias, one batch of short sentences
        {"name": "train f16 odd", "op": "train", "dtype": "f16", "B": 13, "K": 1, "L": 37, "H": 331, "V": 9999,
         "bias": False, "pad": True, "banned": 0, "cut": True},
        # log p(x|z) of a chunk of the importance-weighted estimate: 4 sentences, 64 latent samples of each
        {"name": "seq bf16 4x64x64", "op": "seq", "dtype": "bf16", "B": 4, "K": 64, "L": 64, "H": 768, "V": 50265,
         "bias": True, "pad": True, "banned": 3, "cut": False},
        # the same in 32 bits, 2 sentences
        {"name": "seq f32 2x32x64", "op": "seq", "dtype": "f32", "B": 2, "K": 32, "L": 64, "H": 768, "V": 50265,
         "bias": True, "pad": True, "banned": 3, "cut": False},
        # scoring the next token of one running sequence: latency counts
        {"name": "token bf16 1", "op": "token", "dtype": "bf16", "B": 1, "K": 1, "L": 1, "H": 768, "V": 50265,
         "bias": True, "pad": False, "banned": 2, "cut": False},
        # the next token of a batch of running sequences, in 32 bits
        {"name": "token f32 24", "op": "token", "dtype": "f32", "B": 24, "K": 1, "L": 1, "H": 768, "V": 50265,
         "bias": True, "pad": False, "banned": 0, "cut": False},
        # gradients of the latent heads and a small decoder, in one buffer, within the bound: nothing to scale
        {"name": "clip f32 small", "op": "clip", "dtype": "f32", "out": "", "layers": 2, "width": 100, "vocab": 999,
         "scale": 0.5},
        # an encoder and decoder of 8 layers, 16-bit gradients clipped into the optimizer's 32-bit buffer
        {"name": "clip bf16 to f32", "op": "clip", "dtype": "bf16", "out": "f32", "layers": 16, "width": 512,
         "vocab": 50265, "scale": 2.0},
        # the largest: 32-bit gradients of a wide model, clipped into a second buffer
        {"name": "clip f32 large", "op": "clip", "dtype": "f32", "out": "f32", "layers": 24, "width": 1024,
         "vocab": 50265, "scale": 3.0},
        # 32-bit gradients in place on a step whose norm is within the bound, as most steps are
        {"name": "clip f32 within", "op": "clip", "dtype": "f32", "out": "", "layers": 12, "width": 640,
         "vocab": 32000, "scale": 0.9},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["train", "train", "seq", "token", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op == "clip":
        out = rng.choice(["", "", "f32"])
        return {"op": op, "dtype": dtype, "out": out, "layers": _log_int(rng, 1, 24), "width": _log_int(rng, 40, 1000),
                "vocab": _log_int(rng, 500, 50000), "scale": rng.uniform(0.3, 0.95) if not out else rng.uniform(1.5, 9.0)}
    H = rng.choice([_log_int(rng, 48, 1024), 64 * rng.randint(2, 16)])
    case = {"op": op, "dtype": dtype, "B": 1, "K": 1, "L": 1, "H": H, "V": _log_int(rng, 800, 50265),
            "bias": rng.random() < 0.7, "pad": rng.random() < 0.6, "banned": rng.choice([0, 3]), "cut": rng.random() < 0.4}
    if op == "token":
        case |= {"B": _log_int(rng, 1, 64), "pad": False, "cut": False}
    elif op == "seq":
        case |= {"B": _log_int(rng, 1, 8), "K": _log_int(rng, 1, 64), "L": _log_int(rng, 4, 64), "cut": False}
    else:
        case |= {"B": _log_int(rng, 2, 32), "L": _log_int(rng, 4, 256), "banned": 0}
    return case


def _lengths(case):
    """How many tokens of each sentence are there; the others are padding.  One sentence in 16 has none."""
    B, L = case["B"], case["L"]
    if not case["pad"]:
        return [L] * B
    r = random.Random(B * 1000 + L)
    return [0 if i % 16 == 15 else r.randint(max(1, L // 4), L) for i in range(B)]


def _shapes(case):
    w = case["width"]
    layer = [(w, w), (w,), (w, w), (w,), (w, w), (w,), (w, w), (w,), (w,), (w,), (2 * w, w), (2 * w,), (w, 2 * w), (w,), (w,), (w,)]
    return [(case["vocab"], w), (2 * 32, w), (64,), (w, 32)] + layer * case["layers"] + [(case["vocab"],)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "clip":
        shapes = _shapes(case)
        sizes = [math.prod(s) for s in shapes]
        flat = torch.randn(sum(sizes), device=dev, generator=g)
        # one scale for each part, as layers differ in the size of their gradients
        scales = torch.exp(torch.randn(8, device=dev, generator=g)) * 1e-3
        flat *= scales[torch.arange(flat.numel(), device=dev) * 8 // flat.numel()]
        flat = flat.to(dt)
        ends = [0]
        for n in sizes:
            ends.append(ends[-1] + n)
        views = lambda f: [f[a:b].view(s) for a, b, s in zip(ends, ends[1:], shapes)]
        out = torch.empty(flat.numel(), device=dev, dtype=DTYPES[case["out"]]) if case["out"] else None
        norm = float(flat.double().norm())
        return {"op": "clip", "flat": flat, "grads": views(flat), "out_flat": out, "max_norm": norm / case["scale"],
                "outs": None if out is None else views(out)}
    B, K, L, H, V = (case[k] for k in "BKLHV")
    # hidden states as they leave a layer norm; a cut case has one position more, whose successor is not known
    hidden = torch.randn(B, K, L + int(case["cut"]), H, device=dev, generator=g).to(dt)
    hidden = hidden[:, :, :L]
    weight = (torch.randn(V, H, device=dev, generator=g) * (2.0 / math.sqrt(H))).to(dt)
    rank = torch.randperm(V, device=dev, generator=g)
    freq = -torch.log(rank + 1.0)          # words by their rank in the language
    bias = (0.5 * freq).to(dt) if case["bias"] else None
    if case["banned"] and bias is not None:
        bias[:case["banned"]] = -math.inf  # tokens that are never produced
    ids = torch.multinomial(torch.exp(freq), B * L, replacement=True, generator=g).view(B, L)
    ids = ids.clamp_(min=case["banned"])
    lengths = torch.tensor(_lengths(case), device=dev)
    targets = torch.where(torch.arange(L, device=dev) < lengths[:, None], ids, IGNORE)
    if K == 1:
        hidden = hidden[:, 0]
    else:
        targets = targets[:, None].expand(B, K, L)     # every latent sample of a sentence scores the same words
    if case["op"] == "token":
        hidden, targets = hidden[:, 0], targets[:, 0]
    if case["op"] == "train":
        hidden, weight = hidden.detach().requires_grad_(), weight.requires_grad_()
        bias = bias.requires_grad_() if bias is not None else None
    return {"op": case["op"], "hidden": hidden, "weight": weight, "bias": bias, "targets": targets}


def _plain_log_probs(hidden, weight, bias, targets):
    """Log-likelihood of each target (0 where there is none), the shifted exponentials, their sums, the mask."""
    logits = hidden.float() @ weight.float().t()
    if bias is not None:
        logits += bias.float()
    top = logits.amax(-1, keepdim=True)
    there = targets != IGNORE
    at = targets.clamp(min=0)[..., None]
    picked = (logits.gather(-1, at) - top)[..., 0]
    e = logits.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    ll = torch.where(there, picked - total[..., 0].log(), 0.0)
    return ll, e, total, there, at


def _plain_train(hidden, weight, bias, targets):
    h, t = hidden.detach().reshape(-1, hidden.shape[-1]), targets.reshape(-1)
    w, b = weight.detach(), None if bias is None else bias.detach()
    ll, e, total, there, at = _plain_log_probs(h, w, b, t)
    count = there.sum().clamp(min=1).float()
    g = e.mul_(there[:, None] / (total * count))
    g.scatter_add_(1, at, -(there.float() / count)[:, None])
    return {"loss": -ll.sum() / count, "hidden": (g @ w.float()).to(h.dtype).view(hidden.shape), "weight": (g.t() @ h.float()).to(w.dtype),
            "bias": None if b is None else g.sum(0).to(b.dtype)}


def _plain_clip(grads, max_norm, outs):
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()
    coef = (max_norm / (total + 1e-6)).clamp(max=1.0)
    if outs is None:
        [g.mul_(coef) for g in grads]
    else:
        [o.copy_(g.float() * coef) for g, o in zip(grads, outs)]
    return total


def run(state):
    if state["op"] == "clip":
        if own:
            from lvae import grad_ops
            norm = grad_ops.clip_grads(state["grads"], state["max_norm"], out=state["outs"])
        else:
            norm = _plain_clip(state["grads"], state["max_norm"], state["outs"])
        return {"norm": norm, "grads": state["flat"] if state["out_flat"] is None else state["out_flat"]}
    hidden, weight, bias, targets = (state[k] for k in ("hidden", "weight", "bias", "targets"))
    if own:
        from lvae import decoder_ops
        if state["op"] == "seq":
            return decoder_ops.sequence_log_likelihood(hidden, weight, targets, bias=bias, ignore_index=IGNORE)
        if state["op"] == "token":
            return decoder_ops.token_log_likelihood(hidden, weight, targets, bias=bias, ignore_index=IGNORE)
        loss = decoder_ops.vocab_cross_entropy(hidden, weight, targets, bias=bias, ignore_index=IGNORE, reduction="mean")
        grads = torch.autograd.grad(loss, [hidden, weight] + ([] if bias is None else [bias]))
        return {"loss": loss.detach(), "hidden": grads[0], "weight": grads[1], "bias": None if bias is None else grads[2]}
    if state["op"] == "train":
        return _plain_train(hidden, weight, bias, targets)
    ll = _plain_log_probs(hidden, weight, bias, targets)[0]
    return ll.sum(-1, dtype=torch.float64).float() if state["op"] == "seq" else ll


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        more = (torch.finfo(DTYPES[case["out"]]).bits // 8) if case["out"] else 0
        return {"bytes": n * (size + more), "flops": 2 * n}
    kept = sum(_lengths(case)) * case["K"]
    H, V = case["H"], case["V"]
    params = (V * H + (V if case["bias"] else 0)) * size
    ids = 8 * case["B"] * case["L"]
    if case["op"] == "train":   # the logits' product and the two of the gradients
        return {"bytes": 2 * params + (kept + case["B"] * case["L"]) * H * size + ids, "flops": 6 * kept * V * H}
    return {"bytes": params + kept * H * size + ids, "flops": 2 * kept * V * H}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        x = s["flat"].double()
        norm = torch.linalg.vector_norm(x)
        factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": x.mul_(factor)}
    hidden, weight, targets = s["hidden"].detach(), s["weight"].detach().double(), s["targets"]
    V, H = weight.shape
    bias = torch.zeros(V, device=weight.device, dtype=torch.float64) if s["bias"] is None else s["bias"].detach().double()
    flat, ids = hidden.reshape(-1, H), targets.reshape(-1)
    ll = torch.zeros(ids.numel(), device=weight.device, dtype=torch.float64)
    d_hidden, d_weight, d_bias = torch.zeros(flat.shape, device=weight.device, dtype=torch.float64), torch.zeros_like(weight), torch.zeros_like(bias)
    rows = (ids != IGNORE).nonzero()[:, 0]
    n = max(1, rows.numel())
    for some in rows.split(1024):
        x, y = flat[some].double(), ids[some]
        logp = torch.log_softmax(torch.addmm(bias, x, weight.T), dim=1)
        ll[some] = logp[torch.arange(len(some), device=y.device), y]
        if case["op"] == "train":
            diff = logp.exp() - torch.nn.functional.one_hot(y, V)
            d_hidden[some] = diff @ weight / n
            d_weight += diff.T @ x / n
            d_bias += diff.sum(0) / n
    if case["op"] == "train":
        return {"loss": -ll.sum() / n, "hidden": d_hidden.view(hidden.shape), "weight": d_weight, "bias": None if s["bias"] is None else d_bias}
    return ll.view(targets.shape).sum(-1) if case["op"] == "seq" else ll.view(targets.shape)
