"""Cases of the language-model operators: the vocabulary head's cross entropy, its gradient, the same loss for a
virtual-LoRA population, and clipping by the global gradient norm.

`run` computes a case's operator in its plain form (elementary torch operations in 32 bits) or, where `own` is
true, through this package's own operators.
"""

import math
import random

import torch

own = False

IGNORE = -100  # the label of a token that does not count (padding, a prompt)
RANK = 8  # rank of the virtual-LoRA factors
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # scoring a few short rows with a small head: latency
        {"name": "loss_small", "kind": "loss", "rows": 64, "hidden": 256, "vocab": 1000, "dtype": "bf16", "bias": True},
        # the likelihood of one token under a full vocabulary: the weight is read once for a single row
        {"name": "loss_one_token", "kind": "loss", "rows": 1, "hidden": 4096, "vocab": 32000, "dtype": "bf16", "bias": False},
        # perplexity over a long packed batch
        {"name": "loss_large", "kind": "loss", "rows": 16384, "hidden": 4096, "vocab": 131072, "dtype": "bf16", "bias": False},
        # a training step of a toy model with a biased head, one row more than a tile
        {"name": "step_small", "kind": "step", "rows": 129, "hidden": 512, "vocab": 1009, "dtype": "bf16", "bias": True, "mean": True},
        # a padded batch with a vocabulary of no round size, in half precision with a summed loss
        {"name": "step_odd_fp16", "kind": "step", "rows": 1003, "hidden": 1000, "vocab": 50021, "dtype": "fp16", "bias": False, "mean": False},
        # an ordinary micro-batch
        {"name": "step_medium", "kind": "step", "rows": 2048, "hidden": 2048, "vocab": 32768, "dtype": "bf16", "bias": False, "mean": True},
        # a large micro-batch with a large vocabulary
        {"name": "step_large", "kind": "step", "rows": 8192, "hidden": 4096, "vocab": 131072, "dtype": "bf16", "bias": False, "mean": True},
        # the fitness of a handful of individuals
        {"name": "population_small", "kind": "population", "pop": 8, "batch": 64, "hidden": 256, "vocab": 1000, "bias": True},
        # one evaluation of an evolution strategy over a language-model head
        {"name": "population_large", "kind": "population", "pop": 128, "batch": 64, "hidden": 4096, "vocab": 32000, "bias": False},
        # the gradient blocks of a three-layer network: latency
        {"name": "clip_small", "kind": "clip", "tensors": 6, "total": 197376, "dtype": "fp32", "clips": True},
        # hundreds of blocks of all sizes, back to back in one flat gradient
        {"name": "clip_ragged", "kind": "clip", "tensors": 301, "total": 50000017, "dtype": "bf16", "clips": True},
        # the gradient of a large network in 32 bits
        {"name": "clip_large", "kind": "clip", "tensors": 64, "total": 536870912, "dtype": "fp32", "clips": True},
    ]


def draw(rng):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["loss", "step", "step", "population", "clip"])
    if kind == "clip":
        total = size(1000, 500_000_000)
        return {"kind": kind, "tensors": size(1, min(400, total // 100)), "total": total, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "clips": rng.random() < 0.75}
    if kind == "population":
        batch = rng.choice([64, 128])
        return {"kind": kind, "pop": 2 * size(1, 64 * 64 // batch), "batch": batch, "hidden": 128 * size(1, 32), "vocab": size(500, 32000),
                "bias": rng.random() < 0.5}
    hidden = size(64, 4096)
    if rng.random() < 0.8:
        hidden = (hidden + 7) // 8 * 8
    case = {"kind": kind, "rows": size(1, 16384 if kind == "loss" else 8192), "hidden": hidden, "vocab": size(500, 131072),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "bias": rng.random() < 0.3}
    if kind == "step":
        case["mean"] = case["dtype"] == "bf16" and rng.random() < 0.7  # a mean's gradients leave the range of fp16
    return case


def _sizes(case):
    """Element counts of the gradient blocks: spread over a factor of a thousand, an empty one among many."""
    n, total = case["tensors"], case["total"]
    rng = random.Random(1000003 * n + total)
    weights = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(n)]
    if n > 16:
        weights[n // 2] = 0.0
    scale = total / sum(weights)
    sizes = [int(w * scale) for w in weights]
    sizes[0] += total - sum(sizes)
    return sizes


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "clip":
        dtype, total = DTYPES[case["dtype"]], case["total"]
        flat = torch.empty(total, dtype=torch.float32, device=dev).normal_(generator=gen)
        flat = flat.mul_(4.0 / math.sqrt(total)).to(dtype)  # a norm of about 4
        return {"case": case, "flat": flat, "grads": list(flat.split(_sizes(case))), "max_norm": 1.0 if case["clips"] else 100.0}
    hidden, vocab = case["hidden"], case["vocab"]
    bias = torch.randn(vocab, generator=gen, device=dev) * 0.1 if case["bias"] else None
    if case["kind"] == "population":
        pop, batch = case["pop"], case["batch"]
        h = torch.randn(pop, batch, hidden, generator=gen, device=dev).relu().bfloat16()
        w = (torch.randn(vocab, hidden, generator=gen, device=dev) / math.sqrt(hidden)).bfloat16()
        seeds = torch.randint(0, 2**31, (pop,), generator=gen, device=dev)
        labels = torch.randint(0, vocab, (batch,), generator=gen, device=dev)
        labels[torch.rand(batch, generator=gen, device=dev) < 0.1] = IGNORE
        counter = 40
        return {"case": case, "h": h, "w": w, "bias": bias, "seeds": seeds, "labels": labels, "sigma": 0.02, "counter": counter,
                "bias_counter": None if bias is None else counter + (RANK * hidden + RANK * vocab + 3) // 4 * 4}
    dtype, rows = DTYPES[case["dtype"]], case["rows"]
    w = torch.randn(vocab, hidden, generator=gen, device=dev) * (1.3 / math.sqrt(hidden))
    labels = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
    h = torch.randn(rows, hidden, generator=gen, device=dev)
    # a trained model gives some tokens' labels a high probability: their hidden state leans towards the label's row
    h += w[labels] * (torch.rand(rows, 1, generator=gen, device=dev) * 6.0)
    if rows > 1:
        labels[torch.rand(rows, generator=gen, device=dev) < 0.1] = IGNORE
        labels[0] = vocab - 1
    return {"case": case, "h": h.to(dtype), "w": w.to(dtype), "bias": bias, "labels": labels}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"loss": _own_loss, "step": _own_step, "population": _own_population, "clip": _own_clip}[kind](state)
    return {"loss": _plain_loss, "step": _plain_step, "population": _plain_population, "clip": _plain_clip}[kind](state)


# ---- the framework's operators -------------------------------------------------------------------------------


def _own_loss(s):
    from evox_b200.loss_kernels import linear_cross_entropy

    return linear_cross_entropy(s["h"], s["w"], s["labels"], s["bias"], ignore_index=IGNORE, reduction="none")


def _own_step(s):
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    return linear_cross_entropy_grad(s["h"], s["w"], s["labels"], s["bias"], ignore_index=IGNORE,
                                     reduction="mean" if s["case"]["mean"] else "sum")


def _own_population(s):
    from evox_b200.lora_kernels import lora_layer_cross_entropy

    return lora_layer_cross_entropy(s["h"], s["w"], s["seeds"], s["counter"], s["sigma"], s["labels"], bias=s["bias"],
                                    bias_counter=s["bias_counter"], ignore_index=IGNORE)


def _own_clip(s):
    from evox_b200.grad_kernels import clip_grad_norm_

    return clip_grad_norm_(s["grads"], s["max_norm"]), s["flat"]


# ---- plain forms ---------------------------------------------------------------------------------------------


def _plain_log_softmax_at(z, labels):
    """(log sum exp, loss) of every row of `z`; the loss of an ignored row is 0."""
    top = z.amax(dim=1, keepdim=True)
    lse = (z - top).exp().sum(dim=1).log() + top[:, 0]
    valid = labels != IGNORE
    at = z.gather(1, torch.where(valid, labels, 0)[:, None])[:, 0]
    return lse, torch.where(valid, lse - at, 0.0), valid


def _plain_logits(s):
    z = s["h"].float() @ s["w"].float().t()
    return z if s["bias"] is None else z.add_(s["bias"])


def _plain_loss(s):
    return _plain_log_softmax_at(_plain_logits(s), s["labels"])[1]


def _plain_step(s):
    labels = s["labels"]
    z = _plain_logits(s)
    lse, loss, valid = _plain_log_softmax_at(z, labels)
    weight = valid / valid.sum() if s["case"]["mean"] else valid.float()
    p = z.sub_(lse[:, None]).exp_()
    p.scatter_add_(1, torch.where(valid, labels, 0)[:, None], torch.full_like(p[:, :1], -1.0))
    p.mul_(weight[:, None])
    dh = (p @ s["w"].float()).to(s["h"].dtype)
    dw = (p.t() @ s["h"].float()).to(s["w"].dtype)
    return (loss * weight).sum(), dh, dw, None if s["bias"] is None else p.sum(dim=0)


def _plain_philox_normal(seeds, n, counter):
    """(len(seeds), n) normals of the Philox4x32-10 streams keyed by `seeds`, from position `counter` on."""
    mask = 0xFFFFFFFF

    def mul(m, c):  # high and low 32 bits of m * c
        return (m * (c >> 16) + (m * (c & 0xFFFF) >> 16)) >> 16, (m * c) & mask

    calls = (n + 3) // 4
    c0 = ((counter + torch.arange(calls, device=seeds.device)) & mask)[None, :].expand(len(seeds), calls)
    c1 = torch.full_like(c0, (counter >> 32) & mask)
    c2 = c3 = torch.zeros_like(c0)
    k0, k1 = (seeds & mask)[:, None], ((seeds >> 32) & mask)[:, None]
    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    u = (torch.stack([c0, c1, c2, c3], dim=2) >> 8).float() * 2.0**-24
    r = torch.sqrt(-2.0 * torch.log(u[:, :, 0::2].clamp(min=1e-10)))
    a = 2.0 * math.pi * u[:, :, 1::2]
    return torch.stack([r * torch.cos(a), r * torch.sin(a)], dim=3).reshape(len(seeds), 4 * calls)[:, :n]


def _plain_population(s):
    h, w, seeds, sigma = s["h"].float(), s["w"].float(), s["seeds"], s["sigma"]
    (pop, batch, hidden), vocab = h.shape, w.shape[0]
    a = _plain_philox_normal(seeds, RANK * hidden, s["counter"]).view(pop, RANK, hidden)
    b = _plain_philox_normal(seeds, RANK * vocab, s["counter"] + (RANK * hidden + 3) // 4 * 4).view(pop, vocab, RANK)
    z = torch.baddbmm(h @ w.t(), h @ a.transpose(1, 2), b.transpose(1, 2), alpha=sigma)
    if s["bias"] is not None:
        z = z + (s["bias"] + sigma * _plain_philox_normal(seeds, vocab, s["bias_counter"]))[:, None, :]
    labels = s["labels"].expand(pop, batch).reshape(-1)
    return _plain_log_softmax_at(z.view(pop * batch, vocab), labels)[1].view(pop, batch)


def _plain_clip(s):
    flat = s["flat"]
    norm = flat.double().square().sum().sqrt().float()
    flat.copy_(flat.float() * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0))
    return norm, flat


# ---- what the operators cannot do without ----------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "clip":
        size, total = (4 if case["dtype"] == "fp32" else 2), case["total"]
        # every gradient is read once; it is written once where it is scaled
        return {"bytes": total * size * (2 if case["clips"] else 1) + 4, "flops": total * (3 if case["clips"] else 2)}
    hidden, vocab = case["hidden"], case["vocab"]
    rows = case["rows"] if kind != "population" else case["pop"] * case["batch"]
    product, operands = 2 * rows * vocab * hidden, 2 * (rows + vocab) * hidden + (4 * vocab if case["bias"] else 0)
    if kind == "loss":
        return {"bytes": operands + 12 * rows, "flops": product}
    if kind == "step":  # logits, gradient of the hidden states, gradient of the weight
        return {"bytes": 2 * operands + 8 * rows + 4, "flops": 3 * product}
    return {"bytes": operands + 8 * (case["pop"] + case["batch"]) + 4 * rows, "flops": product + 2 * rows * RANK * (hidden + vocab)}


# ---- 64-bit values from the definitions -----------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        wide = state["flat"].to(torch.float64)
        norm = torch.linalg.vector_norm(wide)
        factor = min(1.0, state["max_norm"] / (float(norm) + 1e-6))
        return norm, wide * factor
    labels, w = state["labels"], state["w"].double()
    if kind == "population":
        return _exact_population(state, w)
    h = state["h"].double()
    rows, vocab = h.shape[0], w.shape[0]
    keep = labels.ne(IGNORE)
    count = int(keep.sum())
    scale = (1.0 / count if count else math.nan) if case.get("mean") else 1.0
    loss = torch.zeros(rows, dtype=torch.float64, device=h.device)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    db = torch.zeros(vocab, dtype=torch.float64, device=h.device)
    step = max(1, 2**29 // vocab)  # rows at a time: 4 GiB of logits
    for at in range(0, rows, step):
        part = slice(at, at + step)
        logits = torch.mm(h[part], w.t())
        if state["bias"] is not None:
            logits += state["bias"].double()
        index = torch.nonzero(keep[part])[:, 0]
        target = labels[part][index]
        logp = torch.log_softmax(logits, dim=1)
        loss[part][index] = -logp[index, target]
        if kind == "loss":
            continue
        delta = logp.exp()
        delta[index, target] -= 1.0
        delta[~keep[part]] = 0.0
        delta *= scale
        dh[part] = torch.mm(delta, w)
        dw += torch.mm(delta.t(), h[part])
        db += delta.sum(dim=0)
    if kind == "loss":
        return loss
    return loss.sum() * scale, dh, dw, None if state["bias"] is None else db


def _exact_normals(seeds, n, counter):
    """The same streams in 64-bit arithmetic, the generator's products by 16-bit halves of both factors."""
    low = (1 << 32) - 1
    count = -(-n // 4)

    def product(x, constant):
        p, q, r, t = x >> 16, x & 65535, constant >> 16, constant & 65535
        middle = p * t + ((q * t) >> 16)
        other = q * r + (middle & 65535)
        return p * r + (middle >> 16) + (other >> 16), ((other & 65535) << 16) | (q * t & 65535)

    zero = torch.zeros(len(seeds), count, dtype=torch.int64, device=seeds.device)
    words = [zero + ((torch.arange(count, device=seeds.device) + counter) & low), zero + ((counter >> 32) & low), zero, zero]
    for turn in range(10):
        key = [(seeds + turn * 0x9E3779B9) & low, ((seeds >> 32) + turn * 0xBB67AE85) & low]
        (ah, al), (bh, bl) = product(words[0], 0xD2511F53), product(words[2], 0xCD9E8D57)
        words = [bh ^ words[1] ^ key[0][:, None], bl, ah ^ words[3] ^ key[1][:, None], al]
    out = torch.empty(len(seeds), 4 * count, dtype=torch.float64, device=seeds.device)
    for pair in (0, 2):
        first, second = ((words[pair + i] >> 8).double() / 2**24 for i in (0, 1))
        radius = (-2.0 * first.clamp(min=1e-10).log()).sqrt()
        out[:, pair::4], out[:, pair + 1 :: 4] = radius * torch.cos(second * (2 * math.pi)), radius * torch.sin(second * (2 * math.pi))
    return out[:, :n]


def _exact_population(state, w):
    pop, batch, hidden = state["h"].shape
    vocab, counter = w.shape[0], state["counter"]
    keep = state["labels"].ne(IGNORE)
    loss = torch.zeros(pop, batch, dtype=torch.float64, device=w.device)
    for i in range(pop):  # an individual at a time: its own weight, W + sigma B A
        key, h = state["seeds"][i : i + 1], state["h"][i].double()
        a = _exact_normals(key, RANK * hidden, counter).view(RANK, hidden)
        b = _exact_normals(key, RANK * vocab, counter + -(-RANK * hidden // 4) * 4).view(vocab, RANK)
        logits = h @ w.t() + state["sigma"] * ((h @ a.t()) @ b.t())
        if state["bias"] is not None:
            logits += state["bias"].double() + state["sigma"] * _exact_normals(key, vocab, state["bias_counter"])[0]
        logp = torch.log_softmax(logits, dim=1)
        loss[i, keep] = -logp[keep, state["labels"][keep]]
    return loss
