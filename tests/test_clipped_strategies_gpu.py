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


class Recorder:
    """The library, with the workspace addresses of the gradient's calls written down."""

    def __init__(self, lib):
        self._lib, self.workspaces = lib, []

    def __getattr__(self, name):
        fn = getattr(self._lib, name)
        if name != "evox_lora_gradient_tc":
            return fn
        return lambda *a: (self.workspaces.append(a[11]), fn(*a))[1]


@gpu
def test_gradients_under_way_at_once_share_no_workspace(cuda, monkeypatch):
    """Two streams, and a captured call next to eager ones: the operand pieces of one must not land on another's."""
    from evox_b200 import _cabi
    from evox_b200.lora_kernels import lora_gradient_from_seeds

    g = torch.Generator().manual_seed(0)
    fitness = [torch.randn(64, generator=g).to(cuda) for _ in range(3)]
    seeds = [torch.arange(64).to(cuda) + 1000 * i for i in range(3)]

    def gradient(i):
        return lora_gradient_from_seeds(fitness[i], seeds[i], (512, 1024), 8, 40, 64, 0.1)

    want = [gradient(i) for i in range(3)]
    torch.cuda.synchronize()
    recorder = Recorder(_cabi.lib)
    monkeypatch.setattr(_cabi, "lib", recorder)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(gradient(i))
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            assert torch.equal(x, y)
    first, second = set(recorder.workspaces[0::2]), set(recorder.workspaces[1::2])
    assert not first & second
    graph = torch.cuda.CUDAGraph()
    recorder.workspaces.clear()
    with torch.cuda.graph(graph):
        captured = gradient(2)
    with torch.cuda.stream(streams[0]):
        eager = gradient(0)
    graph.replay()
    torch.cuda.synchronize()
    assert recorder.workspaces[0] != recorder.workspaces[1]
    assert torch.equal(captured, want[2]) and torch.equal(eager, want[0])


@gpu
def test_clipped_updates_on_two_streams(cuda):
    from evox_b200.algorithms import VirtualLoRAES

    shapes = [(256, 512), (5,), (512, 256)]
    dim = sum(int(torch.tensor(s).prod()) for s in shapes)
    g = torch.Generator().manual_seed(0)
    centers = [torch.randn(dim, generator=g).to(cuda) for _ in range(2)]
    fits = [torch.randn(32, generator=g).to(cuda) for _ in range(2)]
    seeds = [(torch.arange(32) + 100 * i).to(cuda) for i in range(2)]

    def strategy(i):
        algo = VirtualLoRAES(shapes, 8, 32, centers[i], 0.1, 0.05, device=cuda, max_grad_norm=0.5)
        algo.evaluate = lambda payload: fits[i]
        return algo

    serial = [strategy(i) for i in range(2)]
    for i, algo in enumerate(serial):
        for _ in range(3):
            algo.step(seeds[i])
    torch.cuda.synchronize()
    streams, both = [torch.cuda.Stream() for _ in range(2)], [strategy(i) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for i, algo in enumerate(both):
            with torch.cuda.stream(streams[i]):
                algo.step(seeds[i])
    torch.cuda.synchronize()
    for x, y in zip(serial, both):
        assert torch.equal(x.center, y.center) and torch.equal(x.grad_norm, y.grad_norm)
