"""The first call of a process or of a thread to a tensor-core kernel, inside a capture too: nothing may be set up on that
occasion that a capture does not allow. Every case is a process of its own."""
import subprocess
import sys
from pathlib import Path

import pytest

gpu = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PRELUDE = """
import threading
import torch

from evox_b200.grad_kernels import clip_grad_norm_
from evox_b200.lora_kernels import lora_gradient_from_seeds, lora_layer_bf16, lora_layer_cross_entropy
from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

g = torch.Generator().manual_seed(0)
h, w = torch.randn(100, 64, generator=g).cuda(), torch.randn(300, 64, generator=g).cuda() / 8
labels = torch.randint(0, 300, (100,), generator=g).cuda()
people, layer = torch.randn(2, 64, 256, generator=g).cuda().bfloat16(), torch.randn(256, 256, generator=g).cuda().bfloat16() / 16
seeds, words = torch.arange(2).cuda(), torch.randint(0, 256, (64,), generator=g).cuda()
fitness, many = torch.randn(16, generator=g).cuda(), torch.arange(16).cuda()
half = [t.half().requires_grad_() for t in (h, w)]
bf = [t.bfloat16() for t in (h, w)]


def flat(out):
    return [t for t in (out if isinstance(out, (tuple, list)) else [out]) if t is not None]
"""

CALLS = {
    "loss": "linear_cross_entropy(*bf, labels)",
    "one_row": "linear_cross_entropy(bf[0][:1], bf[1], labels[:1])",
    "gradient": "linear_cross_entropy_grad(*bf, labels)",
    "backward": "torch.autograd.grad(linear_cross_entropy(*half, labels), half)",
    "population": "lora_layer_cross_entropy(people, layer, seeds, 0, 0.05, words)",
    "layer": "lora_layer_bf16(people, layer, seeds, 0, 0.05)",
    "population_gradient": "lora_gradient_from_seeds(fitness, many, (128, 256), 8, 0, 16, 0.1)",
    "clip": "clip_grad_norm_([h.clone(), w.clone()], 1.0)",
}

CAPTURE = """
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = flat({call})
graph.replay()
for x, y in zip(got, flat({call})):
    assert torch.equal(x, y)
"""

THREAD = """
got = []
worker = threading.Thread(target=lambda: got.extend(flat({call})))
worker.start()
worker.join()
torch.cuda.synchronize()
assert got
for x, y in zip(got, flat({call})):
    assert torch.equal(x, y)
"""


@gpu
@pytest.mark.parametrize("form", [CAPTURE, THREAD], ids=["capture", "thread"])
@pytest.mark.parametrize("name", CALLS)
def test_first_call(cuda, name, form):
    code = PRELUDE + form.format(call=CALLS[name])
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
