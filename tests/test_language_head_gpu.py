"""The vocabulary head of a virtual-LoRA population, the problem and the strategies that use it, and clipped updates.

Bound of the population's losses, before any run: the regenerated normals are within 2e-6 of the definition's; with
t = h A^T that moves a logit by sigma sum_q (2e-6 |t_q| + (2e-6 + 2^-20 sqrt(k)) sum |h| |b_q|) and sigma 2e-6 for the
bias noise; the product adds (k / 16 + 8) 2^-23 sum |h w|; loss: twice a row's largest logit error
plus 2^-21 (max |z| + 16), as for the plain head."""
import pytest
import torch
from torch import nn

from oracle import lora

gpu = pytest.mark.gpu
IGNORE = -100


def population(pop, batch, k, vocab, bias, seed=0):
    g = torch.Generator().manual_seed(seed + pop * 31 + vocab)
    h = torch.randn(pop, batch, k, generator=g).relu().bfloat16()
    w = (torch.randn(vocab, k, generator=g) / k**0.5).bfloat16()
    seeds = torch.randint(0, 2**31, (pop,), generator=g, dtype=torch.int64)
    labels = torch.randint(0, vocab, (batch,), generator=g)
    labels[torch.rand(batch, generator=g) < 0.2] = IGNORE
    labels[0], labels[-1] = vocab - 1, 0
    return h, w, seeds, labels, torch.randn(vocab, generator=g) * 0.2 if bias else None


def wanted(h, w, seeds, labels, bias, counter, bias_counter, sigma):
    """(losses, bounds) in 64 bits."""
    pop, batch, k = h.shape
    a, b = lora.generate_lora_factors(seeds, (w.shape[0], k), 8, counter)
    h, w, a, b = (x.double().cuda() for x in (h, w, a, b))
    t = h @ a.transpose(1, 2)
    z = h @ w.t() + sigma * (t @ b.transpose(1, 2))
    if bias is not None:
        z += bias.double().cuda()
        if bias_counter is not None:
            z += sigma * lora.generate_lora_factors(seeds, (w.shape[0],), 8, bias_counter).double().cuda()[:, None]
    move = sigma * (2e-6 * t.abs().sum(dim=2, keepdim=True)
                    + (2e-6 + 2.0**-20 * k**0.5) * h.abs().sum(dim=2, keepdim=True) * b.abs().sum(dim=2)[:, None]
                    + 2e-6) + (k / 16 + 8) * 2.0**-23 * (h.abs() @ w.abs().t())
    tol = 2 * move.amax(dim=2) + 2.0**-21 * (z.abs().amax(dim=2) + 16)
    y = labels.cuda()
    valid = y != IGNORE
    loss = torch.logsumexp(z, dim=2) - z.gather(2, torch.where(valid, y, 0).expand(pop, batch)[:, :, None])[:, :, 0]
    return torch.where(valid, loss, 0.0), tol


@gpu
@pytest.mark.parametrize("pop,batch,k,vocab,bias", [
    (2, 64, 128, 1, False), (2, 64, 128, 5, True), (1, 128, 256, 256, True), (3, 128, 256, 300, True), (6, 64, 512, 1000, False),
    (8, 64, 512, 1009, True), (4, 128, 128, 4133, True), (64, 64, 256, 515, False)])
def test_population_loss(cuda, pop, batch, k, vocab, bias):
    from evox_b200.lora_kernels import lora_layer_cross_entropy, raise_on_kernel_errors

    h, w, seeds, labels, b = population(pop, batch, k, vocab, bias)
    for sigma, bias_counter in ((0.05, 4096 if bias else None), (0.0, None)):
        want, tol = wanted(h, w, seeds, labels, b, 40, bias_counter, sigma)
        got = lora_layer_cross_entropy(h.cuda(), w.cuda(), seeds.cuda(), 40, sigma, labels.cuda(), bias=None if b is None else b.cuda(),
                                       bias_counter=bias_counter)
        assert got.shape == (pop, batch) and got.dtype == torch.float32
        off = (got.double() - want).abs() - tol
        assert bool((off <= 0).all()), float(off.max())
        assert bool((got[:, (labels == IGNORE).cuda()] == 0).all())
    raise_on_kernel_errors()


@gpu
def test_population_loss_with_a_given_projection_and_odd_labels(cuda):
    from evox_b200.lora_kernels import lora_layer_bf16, lora_layer_cross_entropy

    h, w, seeds, labels, _ = population(4, 64, 256, 777, False)
    args = h.cuda(), w.cuda(), seeds.cuda(), 40, 0.05
    alone = lora_layer_cross_entropy(*args, labels.cuda())
    a, _ = lora.generate_lora_factors(seeds, (777, 256), 8, 40)
    given = lora_layer_cross_entropy(*args, labels.cuda(), t=(h.float() @ a.transpose(1, 2)).cuda())
    want, tol = wanted(h, w, seeds, labels, None, 40, None, 0.05)
    assert bool(((given.double() - want).abs() <= tol).all())
    for bad in (777, 800, -1, 2**40):
        y = labels.clone()
        y[5] = bad
        got = lora_layer_cross_entropy(*args, y.cuda())
        keep = torch.arange(64) != 5
        assert bool(torch.isnan(got[:, 5]).all()) and torch.equal(got[:, keep], alone[:, keep])
    graph = torch.cuda.CUDAGraph()
    static = labels.cuda()
    with torch.cuda.graph(graph):
        out = lora_layer_cross_entropy(*args, static)
    graph.replay()
    assert torch.equal(out, alone)
    # a projected layer before it, as the problem chains them
    y, t_next = lora_layer_bf16(h.cuda(), torch.eye(256).bfloat16().cuda(), seeds.cuda(), 9000, 0.0, relu=True, next_counter=40)
    assert bool(((lora_layer_cross_entropy(y, w.cuda(), seeds.cuda(), 40, 0.05, labels.cuda(), t=t_next).double() - want).abs() <= tol).all())


def head_problem(vocab, bias, criterion, compute_dtype, device, pop=4, batch=64, width=256, reduction="mean", lead=True):
    from evox_b200.problems import VirtualLoRAProblem

    g = torch.Generator().manual_seed(vocab)
    layers = [nn.Linear(width, width, bias=bias), nn.ReLU(), nn.Linear(width, vocab, bias=bias)]
    layers = layers if lead else layers[2:]
    with torch.no_grad():
        for p in (p for m in layers for p in m.parameters()):
            p.copy_((torch.randn(p.shape, generator=g) / width**0.5).bfloat16().float())
    model = nn.Sequential(*layers)
    x = torch.randn(pop, batch, width, generator=g).bfloat16()
    labels = torch.randint(0, vocab, (batch,), generator=g)
    labels[3] = IGNORE
    prob = VirtualLoRAProblem(model, [(x, labels)], criterion, 8, device=device, compute_dtype=compute_dtype, reduction=reduction)
    center = torch.cat([p.detach().reshape(-1) for p in model.parameters()]).to(device)
    return prob, center, torch.randint(0, 2**31, (pop,), generator=g, dtype=torch.int64).to(device), x, labels


@gpu
@pytest.mark.parametrize("vocab,bias,lead,reduction", [(512, False, True, "mean"), (777, True, True, "mean"), (1000, True, False, "sum")])
def test_problem_ends_in_the_loss(cuda, vocab, bias, lead, reduction, monkeypatch):
    """The fused head against torch's criterion on the logits the same problem would otherwise store (bf16 hidden layer in
    both; rounding only)."""
    from evox_b200.problems import virtual_lora_problem as module

    prob, center, seeds, x, labels = head_problem(vocab, bias, nn.CrossEntropyLoss(reduction="none"), torch.bfloat16, cuda, lead=lead, reduction=reduction)
    calls = []
    real = module.lora_layer_cross_entropy
    monkeypatch.setattr(module, "lora_layer_cross_entropy", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    got = prob.evaluate((center, seeds, 0.05))
    assert got.shape == (4,) and calls == [1]
    # other criteria (label smoothing) keep the logits: same forward, loss by torch
    logits = prob._virtual_forward(x.to(cuda), center, seeds, 0.05, 4)
    loss = nn.functional.cross_entropy(logits.double().reshape(-1, vocab), labels.to(cuda).repeat(4), reduction="none").view(4, 64)
    want = loss.mean(dim=1) if reduction == "mean" else loss.sum(dim=1)
    # the stored-logits path multiplies the last layer in fp32 where the vocabulary is odd, in bf16 operands otherwise; the
    # weights are bf16 values, so the operands agree and only sums differ
    assert float(((got.double() - want) / want).abs().max()) <= 2e-5
    smooth, *_ = head_problem(vocab, bias, nn.CrossEntropyLoss(reduction="none", label_smoothing=0.1), torch.bfloat16, cuda, lead=lead, reduction=reduction)
    assert smooth.evaluate((center, seeds, 0.05)).shape == (4,) and calls == [1]
    fp32, *_ = head_problem(vocab, bias, nn.CrossEntropyLoss(reduction="none"), torch.float32, cuda, lead=lead, reduction=reduction)
    assert fp32.evaluate((center, seeds, 0.05)).shape == (4,) and calls == [1]


@gpu
@pytest.mark.parametrize("optimizer", [None, "adam"])
def test_clipped_strategy_step(cuda, optimizer):
    """VirtualLoRAES over a cross-entropy head, with and without a bound on the gradient: the clipped step is the update
    with the scaled gradient."""
    from evox_b200.algorithms import VirtualLoRAES
    from evox_b200.grad_kernels import grad_norm
    from evox_b200.lora_kernels import lora_gradient_from_seeds
    from evox_b200.workflows import StdWorkflow

    prob, center, seeds, _, _ = head_problem(777, True, nn.CrossEntropyLoss(reduction="none"), torch.bfloat16, cuda)
    lr, sigma = 0.5, 0.05

    def run(limit):
        algo = VirtualLoRAES(prob.param_shapes, 8, 4, center, lr, sigma, optimizer=optimizer, device=cuda, max_grad_norm=limit)
        wf = StdWorkflow(algo, prob, device=cuda)
        algo.step(seeds)
        return algo, wf

    free, _ = run(None)
    loose, _ = run(1e9)
    assert torch.equal(free.center, loose.center) and free.grad_norm is None
    fitness = prob.evaluate((center, seeds, sigma))
    blocks = [lora_gradient_from_seeds(fitness, seeds, s, 8, o, 4, sigma) for s, o in zip(prob.param_shapes, prob.counter_offsets)]
    norm = float(grad_norm(blocks))
    assert float(loose.grad_norm) == norm
    tight, _ = run(norm / 8)
    grad = torch.cat([b.reshape(-1) for b in blocks]).double() / 8
    moved = center.double() - tight.center.double()
    if optimizer is None:
        # a rounding of the factor's three, the product and the update each, relative to what they round
        assert bool(((moved - lr * grad).abs() <= lr * grad.abs() * 2.0**-20 + center.double().abs() * 2.0**-23 + 1e-9).all())
    else:
        assert float((tight.exp_avg.double() - 0.1 * grad).abs().max()) <= float(grad.abs().max()) * 2.0**-20
    # several generations on end, loss and clipping together
    algo, wf = run(norm / 8)
    for _ in range(3):
        wf.step()
    assert bool(torch.isfinite(algo.center).all()) and float(algo.grad_norm) > 0


@gpu
def test_openes_clips_in_eager_and_traced_steps(cuda):
    from evox_b200.algorithms import OpenES
    from evox_b200.problems.numerical import Sphere
    from evox_b200.workflows import StdWorkflow

    def run(compiled, limit):
        torch.manual_seed(0)
        torch._dynamo.reset()
        algo = OpenES(256, torch.full((64,), 3.0), 0.05, 0.1, device=cuda, max_grad_norm=limit)
        wf = StdWorkflow(algo, Sphere(), device=cuda)
        step = torch.compile(wf.step, backend="aot_eager", fullgraph=True) if compiled else wf.step
        centers = []
        for g in range(3):
            torch.manual_seed(g)
            step()
            centers.append(algo.center.clone())
        return algo, centers

    algo, clipped = run(False, 2.0)
    assert float(algo.grad_norm) > 2.0
    before = torch.full((64,), 3.0, device=cuda)
    assert abs(float((clipped[0] - before).norm()) - 0.05 * 2.0) <= 1e-5
    for x, y in zip(clipped, run(True, 2.0)[1]):
        assert torch.equal(x, y)
    _, free = run(False, None)
    for x, y in zip(free, run(False, 1e9)[1]):
        assert torch.equal(x, y)


@gpu
def test_registered_operators(cuda):
    import evox_b200.ops  # noqa: F401
    from evox_b200 import grad_kernels, lora_kernels, loss_kernels

    o = torch.ops.evox_b200
    h, w, seeds, labels, b = (None if t is None else t.cuda() for t in population(2, 64, 128, 300, True))
    assert torch.equal(o.lora_layer_cross_entropy(h, w, seeds, 40, 0.05, labels, b, 4096, None, IGNORE),
                       lora_kernels.lora_layer_cross_entropy(h, w, seeds, 40, 0.05, labels, bias=b, bias_counter=4096))
    flat = h[0]
    assert torch.equal(o.linear_cross_entropy(flat, w, labels, b, IGNORE, "none"), loss_kernels.linear_cross_entropy(flat, w, labels, b, reduction="none"))
    for x, y in zip(o.linear_cross_entropy_grad(flat, w, labels, b, None, IGNORE, "mean"), loss_kernels.linear_cross_entropy_grad(flat, w, labels, b)):
        assert torch.equal(x, y)
    assert o.linear_cross_entropy_grad(flat, w, labels, None, None, IGNORE, "mean")[3].numel() == 0
    g1 = [torch.randn(100, device=cuda), torch.randn(7, 3, device=cuda)]
    g2 = [t.clone() for t in g1]
    assert torch.equal(o.grad_norm(g1), grad_kernels.grad_norm(g1))
    assert torch.equal(o.clip_grad_norm_(g1, 1.0), grad_kernels.clip_grad_norm_(g2, 1.0)) and all(map(torch.equal, g1, g2))
    torch.library.opcheck(o.linear_cross_entropy.default, (flat, w, labels, b, IGNORE, "mean"), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(o.clip_grad_norm_.default, (g1, 1.0), test_utils=("test_schema", "test_faketensor"))


# ---- host side ------------------------------------------------------------------------------------------------


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import evox_b200.ops  # noqa: F401

    o = torch.ops.evox_b200
    with FakeTensorMode():
        h, w, y, b = torch.empty(10, 64, dtype=torch.bfloat16), torch.empty(99, 64, dtype=torch.bfloat16), torch.empty(10, dtype=torch.int64), torch.empty(99)
        assert o.linear_cross_entropy(h, w, y, b, -100, "mean").shape == () and o.linear_cross_entropy(h, w, y, None, -100, "none").shape == (10,)
        loss, dh, dw, db = o.linear_cross_entropy_grad(h, w, y, b, None, -100, "mean")
        assert dh.shape == h.shape and dw.dtype == torch.bfloat16 and dw.shape == w.shape and db.shape == (99,) and loss.dtype == torch.float32
        hp = torch.empty(2, 64, 128, dtype=torch.bfloat16)
        assert o.lora_layer_cross_entropy(hp, w, torch.empty(2, dtype=torch.int64), 0, 0.1, y, None, None, None, -100).shape == (2, 64)
        assert o.grad_norm([b, h]).shape == () and o.clip_grad_norm_([b], 1.0).dtype == torch.float32


def test_population_refusals():
    from evox_b200 import _cabi
    from evox_b200.lora_kernels import lora_layer_cross_entropy

    h, w = torch.zeros(2, 64, 128, dtype=torch.bfloat16), torch.zeros(9, 128, dtype=torch.bfloat16)
    seeds, y = torch.zeros(2, dtype=torch.int64), torch.zeros(64, dtype=torch.int64)
    for args, kw, said in (((h.float(), w, seeds, 0, 0.1, y), {}, "bf16"), ((h, w[:, :64], seeds, 0, 0.1, y), {}, "shape mismatch"),
                           ((h[0], w, seeds, 0, 0.1, y), {}, "shape mismatch"), ((h, w, seeds[:1], 0, 0.1, y), {}, "seeds"),
                           ((h, w, seeds, 0, 0.1, y[:3]), {}, "labels"), ((h, w, seeds, 0, 0.1, y.int()), {}, "labels"),
                           ((h, w, seeds, 0, 0.1, y), {"bias": torch.zeros(8)}, "bias"), ((h, w, seeds, 0, 0.1, y), {"t": torch.zeros(2, 64, 4)}, "t must"),
                           ((h[:, :48], w, seeds, 0, 0.1, y[:48]), {}, "not supported"), ((h[..., :64], w[:, :64], seeds, 0, 0.1, y), {}, "not supported")):
        with pytest.raises(_cabi.EvoxKernelError, match=said):
            lora_layer_cross_entropy(*args, **kw)
    lib = _cabi.lib
    ok = dict(h=256, w=256, bias=None, t=256, seeds=256, b_counter=0, has=0, nc=0, sigma=0.1, pop=2, batch=64, k=128, vocab=9, r=8, labels=256, ignore=-100,
              loss=256, ws=256, nbytes=1 << 20, err=256, stream=None)

    def call(**kw):
        return lib.evox_lora_cross_entropy_bf16(*{**ok, **kw}.values())

    for kw in (dict(h=None), dict(t=None), dict(labels=None), dict(ws=None), dict(err=None), dict(vocab=0), dict(r=4), dict(k=64), dict(batch=48),
               dict(pop=1), dict(h=264), dict(t=260), dict(ws=264)):
        assert call(**kw) == -1, kw
        assert b"lora_cross_entropy" in lib.evox_last_error()
    assert call(nbytes=8) == -3
    assert lib.evox_lora_cross_entropy_supported(2, 64, 128, 50021, 8) == 1 and lib.evox_lora_cross_entropy_supported(2, 64, 128, 0, 8) == 0


def test_strategies_refuse_bad_bounds():
    from evox_b200.algorithms import OpenES, VirtualLoRAES

    for bad in (0.0, -1.0):
        with pytest.raises(AssertionError, match="max_grad_norm"):
            OpenES(4, torch.zeros(3), 0.1, 0.1, device="cpu", max_grad_norm=bad)
    with pytest.raises(AssertionError, match="shard"):
        VirtualLoRAES([(3,)], 8, 4, torch.zeros(3), 0.1, 0.1, device="cpu", shard=True, max_grad_norm=1.0)
