"""The status word of the tensor-core launches: what a call does while it is set, as it is after a bounded wait expired."""
import pytest
import torch

from tests.test_linear_cross_entropy_gpu import make

gpu = pytest.mark.gpu


@pytest.fixture
def word(cuda):
    """The device's status word; reset and reported afterwards whatever a test did."""
    from evox_b200.lora_kernels import raise_on_kernel_errors, status_word

    raise_on_kernel_errors()
    yield status_word(cuda)
    status_word(cuda).zero_()
    raise_on_kernel_errors()


def population(cuda, pop=4, batch=64, k=256, vocab=700):
    g = torch.Generator().manual_seed(0)
    h = torch.randn(pop, batch, k, generator=g).bfloat16().to(cuda)
    w = (torch.randn(vocab, k, generator=g) / k**0.5).bfloat16().to(cuda)
    return h, w, torch.arange(pop, device=cuda), 0, 0.05, torch.randint(0, vocab, (batch,), generator=g).to(cuda)


@gpu
@pytest.mark.parametrize("rows,hidden,vocab", [(300, 256, 5000), (20, 512, 3000), (1, 2048, 4096), (2000, 2048, 9000)])
def test_launches_end_while_the_word_is_set_and_work_when_it_is_not(cuda, word, rows, hidden, vocab):
    from evox_b200.lora_kernels import lora_layer_cross_entropy
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, b = make(rows, hidden, vocab, torch.bfloat16, True)
    people = population(cuda)

    def run():
        return [linear_cross_entropy(h, w, labels, b, reduction="none"), *linear_cross_entropy_grad(h, w, labels, b), lora_layer_cross_entropy(*people)]

    want = run()
    for code in (1, 3, 4):
        word.fill_(code)
        run()
        torch.cuda.synchronize()
        assert int(word) == code  # the first report stays
    word.zero_()
    for x, y in zip(want, run()):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("rows,hidden,vocab", [(300, 256, 5000), (20, 512, 3000), (1, 2048, 4096), (700, 64, 130)])
def test_results_are_nan_while_the_word_is_set(cuda, word, rows, hidden, vocab):
    """Rows that count and rows that do not; through every form of the call, an eager one after a capture among them."""
    from evox_b200._cabi import EvoxKernelError
    from evox_b200.lora_kernels import lora_layer_cross_entropy, raise_on_kernel_errors
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, b = make(rows, hidden, vocab, torch.bfloat16, True)
    valid = labels != -100
    hs = h.clone().requires_grad_()
    people = population(cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = linear_cross_entropy(h, w, labels, b)
    graph.replay()
    good = float(captured)
    assert torch.isfinite(captured)
    word.fill_(4)
    for reduction in ("none", "sum", "mean"):
        assert bool(torch.isnan(linear_cross_entropy(h, w, labels, b, reduction=reduction)).all())
    for chunk in (None, max(1, rows // 3)):
        loss, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, chunk_rows=chunk)
        assert torch.isnan(loss) and bool(torch.isnan(dh[valid]).all()) and bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all())
    linear_cross_entropy(hs, w, labels, b).backward()
    assert bool(torch.isnan(hs.grad[valid]).all())
    assert bool(torch.isnan(lora_layer_cross_entropy(*people)).all())
    graph.replay()
    assert torch.isnan(captured)
    with pytest.raises(EvoxKernelError, match="status 4"):
        raise_on_kernel_errors()
    graph.replay()
    assert float(captured) == good and bool(torch.isfinite(lora_layer_cross_entropy(*people)).all())


@gpu
def test_a_word_made_in_a_capture_serves_its_replays(cuda, word, monkeypatch):
    from evox_b200 import lora_kernels
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    h, w, labels, b = make(300, 128, 900, torch.bfloat16, True)
    want = linear_cross_entropy_grad(h, w, labels, b)
    monkeypatch.setattr(lora_kernels, "_status_words", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = linear_cross_entropy_grad(h, w, labels, b)
        assert not lora_kernels._status_words
        more = [torch.ones(1, device=cuda) for _ in range(20)]  # may take the word's place
    for _ in range(2):
        graph.replay()
        for x, y in zip(want, got):
            assert torch.equal(x, y)
    assert all(float(m) == 1.0 for m in more)
