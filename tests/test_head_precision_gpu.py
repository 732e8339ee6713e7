"""Vocabulary heads that the bf16 layer kernel does not take keep the digits of their fp32 operands, as before they ended in
the loss.

Bound of a loss, before any run: pieces of bf16 (8 digits each, three of them) leave 2^-24 of |h w|, and pairs below 2^-24 of
the largest are left out (three of them for fp32 activations): 2^-22 sum |h w|; a 32-bit accumulator that may truncate in n k / 16
additions, (n k / 16 + 8) 2^-23 sum |h w|; the correction sigma (2e-6 |t| + (2e-6 + 2^-20 sqrt(k)) sum |h| |b|) and the noise sigma 2e-6;
twice that for a loss, plus 2^-21 (max |z| + 16)."""
import pytest
import torch
from torch import nn

from oracle import lora

gpu = pytest.mark.gpu


def build(vocab, width, bias, lead, activation, x_dtype, device, pop=4, batch=64):
    from evox_b200.problems import VirtualLoRAProblem

    g = torch.Generator().manual_seed(vocab + width)
    head = nn.Linear(width, vocab, bias=bias)
    layers = [nn.Linear(width, width, bias=False), activation(), head] if lead else [head]
    with torch.no_grad():
        for p in (p for m in layers for p in m.parameters()):
            p.copy_(torch.randn(p.shape, generator=g) / width**0.5)  # 24 digits
    model = nn.Sequential(*layers)
    x = torch.randn(pop, batch, width, generator=g).to(x_dtype)
    labels = torch.randint(0, vocab, (batch,), generator=g)
    labels[3] = -100
    prob = VirtualLoRAProblem(model, [(x, labels)], nn.CrossEntropyLoss(reduction="none"), 8, device=device, compute_dtype=torch.bfloat16)
    center = torch.cat([p.detach().reshape(-1) for p in model.parameters()]).to(device)
    return prob, center, torch.randint(0, 2**31, (pop,), generator=g, dtype=torch.int64).to(device), x, labels


@gpu
@pytest.mark.parametrize("vocab,width,bias,lead,activation,x_dtype", [
    (777, 256, True, True, nn.ReLU, torch.bfloat16),    # bf16 activations from the layer before: three pieces of the weight
    (1000, 512, False, True, nn.Tanh, torch.bfloat16),
    (300, 128, True, False, None, torch.float32),       # fp32 inputs: three pieces of both
    (5000, 1024, False, False, None, torch.bfloat16),
])
def test_odd_heads_keep_fp32_digits(cuda, vocab, width, bias, lead, activation, x_dtype, monkeypatch):
    from evox_b200.lora_kernels import raise_on_kernel_errors
    from evox_b200.problems import virtual_lora_problem as module

    prob, center, seeds, x, labels = build(vocab, width, bias, lead, activation, x_dtype, cuda)
    losses = []
    real = module.lora_layer_cross_entropy
    monkeypatch.setattr(module, "lora_layer_cross_entropy", lambda *a, **k: (losses.append(real(*a, **k)), losses[-1])[1])
    sigma = 0.05
    fitness = prob.evaluate((center, seeds, sigma))
    raise_on_kernel_errors()
    assert len(losses) == 1
    # the head's input, from the same problem without its head; the head in 64 bits on the fp32 parameters
    h = x.to(cuda)
    if lead:
        trunk = module.VirtualLoRAProblem(nn.Sequential(*list(prob.model.children())[:2]), [], nn.MSELoss(), 8, device=cuda, compute_dtype=torch.bfloat16)
        h = trunk._virtual_forward(h, center[: width * width], seeds, sigma, 4).bfloat16()  # as a layer passes it on
    h = h.double()
    weight, wi = prob._param(center, f"{len(prob.model) - 1}.weight")
    w = weight.double()
    a, b = (f.double().to(cuda) for f in lora.generate_lora_factors(seeds.cpu(), (vocab, width), 8, prob.counter_offsets[wi]))
    t = h @ a.transpose(1, 2)
    z = h @ w.t() + sigma * (t @ b.transpose(1, 2))
    if bias:
        bias_value, bi = prob._param(center, f"{len(prob.model) - 1}.bias")
        z += bias_value.double() + sigma * lora.generate_lora_factors(seeds.cpu(), (vocab,), 8, prob.counter_offsets[bi]).double().to(cuda)[:, None]
    size = h.abs() @ w.abs().t()
    n = 3 if h.float().bfloat16().double().equal(h) else 6
    move = ((n * width / 16 + 8) * 2.0**-23 + 2.0**-22) * size + sigma * (
        2e-6 * t.abs().sum(dim=2, keepdim=True) + (2e-6 + 2.0**-20 * width**0.5) * h.abs().sum(dim=2, keepdim=True) * b.abs().sum(dim=2)[:, None] + 2e-6)
    tol = 2 * move.amax(dim=2) + 2.0**-21 * (z.abs().amax(dim=2) + 16)
    y = labels.to(cuda)
    valid = y != -100
    want = torch.logsumexp(z, dim=2) - z.gather(2, torch.where(valid, y, 0).expand(4, 64)[:, :, None])[:, :, 0]
    want = torch.where(valid, want, 0.0)
    off = (losses[0].double() - want).abs()
    assert bool((off <= tol).all()), f"{float((off - tol).max())} above the bound, largest error {float(off.max())}"
    # as close as the fp32 kernels, not as bf16 operands: those move a logit by about 2^-9 of |h w|, added in squares
    rounding = 2.0**-9 * torch.sqrt((h**2) @ (w.t() ** 2)).mean()
    assert float(off.mean()) <= 0.05 * float(rounding)
    assert bool(((fitness.double() - want.mean(dim=1)).abs() <= tol.mean(dim=1) + 2.0**-20 * want.mean(dim=1)).all())


def test_pieces_add_up():
    from evox_b200.problems.virtual_lora_problem import _bf16_pieces, _in_bf16_pieces

    g = torch.Generator().manual_seed(0)
    x = torch.randn(1000, generator=g) * torch.exp(torch.randn(1000, generator=g) * 5)
    total = sum(p.double() for p in _bf16_pieces(x))
    assert bool(((total - x.double()).abs() <= x.double().abs() * 2.0**-25).all())
    w = torch.randn(9, 128, generator=g)
    for h in (torch.randn(2, 4, 128, generator=g), torch.randn(2, 4, 128, generator=g).bfloat16()):
        hp, wp = _in_bf16_pieces(h, w)
        assert hp.dtype == wp.dtype == torch.bfloat16 and hp.shape[2] == wp.shape[1] == 128 * (6 if h.dtype == torch.float32 else 3)
        want = h.double() @ w.double().t()
        assert bool(((hp.double() @ wp.double().t() - want).abs() <= 2.0**-22 * (h.double().abs() @ w.double().abs().t())).all())
