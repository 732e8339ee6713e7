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


def test_without_a_bound_there_is_no_norm():
    from evox_b200.algorithms import OpenES

    algo = OpenES(4, torch.zeros(3), 0.1, 0.1, device="cpu")
    assert algo.grad_norm is None and "grad_norm" not in algo.state_dict()
    algo = OpenES(4, torch.zeros(3), 0.1, 0.1, device="cpu", max_grad_norm=1.0)
    assert torch.isnan(algo.grad_norm) and algo.grad_norm.shape == () and "grad_norm" in algo.state_dict()
