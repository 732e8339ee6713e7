"""`max_grad_norm=` of the strategies: the norm that they keep, and the blocks that they clip."""
import pytest
import torch

gpu = pytest.mark.gpu


def sphere(device, limit, pop=256, dim=64):
    from evox_b200.algorithms import OpenES
    from evox_b200.problems.numerical import Sphere
    from evox_b200.workflows import StdWorkflow

    algo = OpenES(pop, torch.full((dim,), 3.0), 0.05, 0.1, device=device, max_grad_norm=limit)
    return algo, StdWorkflow(algo, Sphere(), device=device)


@gpu
def test_grad_norm_is_kept_in_traced_steps(cuda):
    def run(form):
        torch._dynamo.reset()
        algo, wf = sphere(cuda, 2.0)
        traced = torch.compile(wf.step, backend="aot_eager", fullgraph=True)
        norms = []
        for g in range(4):
            torch.manual_seed(g)
            (traced if form == "traced" or (form == "mixed" and g % 2) else wf.step)()
            norms.append(algo.grad_norm.clone())
        return torch.stack(norms)

    want = run("eager")
    assert bool((want > 0).all()) and want.unique().numel() == 4
    assert torch.equal(run("traced"), want) and torch.equal(run("mixed"), want)


@gpu
def test_grad_norm_is_part_of_the_state(cuda):
    from evox_b200.core import use_state, vmap

    algo, wf = sphere(cuda, 2.0)
    assert torch.isnan(algo.grad_norm) and "grad_norm" in algo.state_dict()
    step = use_state(wf.step)
    state = {k: v.clone() for k, v in wf.state_dict().items() if isinstance(v, torch.Tensor)}
    name = next(k for k in state if k.endswith("grad_norm"))
    torch.manual_seed(0)
    new = step(state)
    assert torch.isnan(algo.grad_norm) and float(new[name]) > 0  # the module itself is untouched
    two = {k: torch.stack([v, v]) for k, v in state.items()}
    out = vmap(step, randomness="different")(two)
    assert out[name].shape == (2,) and float(out[name][0]) != float(out[name][1])


@gpu
@pytest.mark.parametrize("optimizer", [None, "adam"])
def test_blocks_behind_one_of_odd_length_are_computed_as_without_a_bound(cuda, optimizer, monkeypatch):
    """A bound that does not bite changes nothing, to the last bit, and stays on the same kernels."""
    from evox_b200 import lora_kernels
    from evox_b200.algorithms import VirtualLoRAES

    shapes = [(3,), (128, 256), (7,), (5, 11), (256, 512), (2,)]
    dim = sum(int(torch.tensor(s).prod()) for s in shapes)
    g = torch.Generator().manual_seed(0)
    center, fitness, seeds = torch.randn(dim, generator=g).to(cuda), torch.randn(16, generator=g).to(cuda), torch.arange(16).to(cuda)
    stored = []
    real = lora_kernels.generate_lora_factors
    monkeypatch.setattr(lora_kernels, "generate_lora_factors", lambda s, shape, *a: (stored.append(tuple(shape)), real(s, shape, *a))[1])

    def run(limit):
        algo = VirtualLoRAES(shapes, 8, 16, center, 0.1, 0.05, optimizer=optimizer, device=cuda, max_grad_norm=limit)
        algo.evaluate = lambda payload: fitness
        stored.clear()
        for _ in range(2):
            algo.step(seeds)
        return algo, list(stored)

    free, without = run(None)
    loose, bounded = run(1e9)
    assert torch.equal(free.center, loose.center) and bounded == without
    assert (128, 256) not in without and (256, 512) not in without
    tight, _ = run(float(loose.grad_norm) / 4)
    assert float(tight.grad_norm) == float(loose.grad_norm)
    if optimizer is None:  # two steps of the quarter gradient; a rounding of the factor's three, the product and each update
        step = (center.double() - free.center.double()) / 4
        moved = center.double() - tight.center.double()
        assert bool(((moved - step).abs() <= step.abs() * 2.0**-20 + 4 * center.double().abs().clamp(min=float(step.abs().max())) * 2.0**-23).all())


def test_without_a_bound_there_is_no_norm():
    from evox_b200.algorithms import OpenES

    algo = OpenES(4, torch.zeros(3), 0.1, 0.1, device="cpu")
    assert algo.grad_norm is None and "grad_norm" not in algo.state_dict()
    algo = OpenES(4, torch.zeros(3), 0.1, 0.1, device="cpu", max_grad_norm=1.0)
    assert torch.isnan(algo.grad_norm) and algo.grad_norm.shape == () and "grad_norm" in algo.state_dict()
