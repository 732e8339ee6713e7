"""`linear_cross_entropy(...).backward()` under upstream gradients that leave the range or the digits of the operands' type,
against the 64-bit formula with the upstream value applied before anything is rounded (bounds: `Formula`)."""
import pytest
import torch

from tests.test_linear_cross_entropy_gpu import Formula, make, near

gpu = pytest.mark.gpu


def backward(h, w, labels, b, reduction, upstream, chunk_rows=None):
    from evox_b200.loss_kernels import linear_cross_entropy

    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2], reduction=reduction, chunk_rows=chunk_rows)
    loss.backward(torch.tensor(upstream, device=h.device))
    return [loss.detach()] + [t.grad for t in leaves]


def near_fp16(got, want, tol, what):
    """As `near`; from 65,520 on (65,504 and half of its step, 32) fp16 has only infinity."""
    over = want.abs() - tol >= 65520
    under = want.abs() + tol < 65520
    assert torch.equal(got.double()[over], torch.sign(want[over]) * torch.inf), what
    near(got[under], want[under], tol[under], what)


@gpu
@pytest.mark.parametrize("rows,hidden,vocab", [(4000, 64, 2000), (40, 64, 300), (129, 100, 1009)])
@pytest.mark.parametrize("upstream", [2.0**16, 2.0**20, 1.0, 1.0 / 3.0])
def test_fp16_mean_under_a_loss_scale(cuda, rows, hidden, vocab, upstream):
    """2^16 is not a number of fp16."""
    h, w, labels, b = make(rows, hidden, vocab, torch.float16, True)
    up = torch.tensor(upstream, device=cuda)
    f = Formula(h, w, labels, b, "mean", up)
    loss, dh, dw, db = backward(h, w, labels, b, "mean", upstream)
    near(loss, f.loss, f.loss_tol, "loss")
    near_fp16(dh, f.dh, f.dh_tol, "dh")
    near_fp16(dw, f.dw, f.dw_tol, "dw")
    near(db, f.db, f.db_tol + 2.0**-22 * f.db.abs(), "db")


@gpu
def test_fp16_gradients_that_only_a_loss_scale_keeps(cuda):
    """dw of a word that is nobody's label and hardly ever predicted is below 2^-25, where fp16 has only 0; under 2^14 it has
    values of 1e-5 to 1e-3."""
    h, w, labels, b = make(2000, 64, 4000, torch.float16, True, ignored=0.0)
    labels = labels % 50
    b[50:] -= 14.0
    f = Formula(h, w, labels, b, "mean", torch.tensor(2.0**14, device=cuda))
    lost = f.dw.abs() < 2.0**-25 * 2.0**14
    assert float(lost.double().mean()) > 0.9
    _, dh, dw, _ = backward(h, w, labels, b, "mean", 2.0**14)
    near(dw, f.dw, f.dw_tol, "dw")
    near(dh, f.dh, f.dh_tol, "dh")
    assert float((dw[lost] != 0).double().mean()) > 0.9


@gpu
def test_fp16_sum_brought_back_into_range_by_the_upstream_gradient(cuda):
    """All rows share a label: its row of dw passes 65,504 in the sum over the rows, not in the mean."""
    rows = 4000
    g = torch.Generator().manual_seed(0)
    h = (20.0 + torch.randn(rows, 64, generator=g)).half().cuda()
    w = (torch.randn(300, 64, generator=g) / 64).half().cuda()
    labels, b = torch.full((rows,), 5, device=cuda), torch.zeros(300, device=cuda)
    f = Formula(h, w, labels, b, "sum", torch.tensor(1.0 / rows, device=cuda))
    assert float(f.dw.abs().max()) * rows > 65504
    _, dh, dw, _ = backward(h, w, labels, b, "sum", 1.0 / rows, chunk_rows=1500)
    near(dw, f.dw, f.dw_tol, "dw")
    near(dh, f.dh, f.dh_tol, "dh")


@gpu
@pytest.mark.parametrize("upstream", [1.0 / 3.0, 1e-3, 12345.678, 2.0**16])
def test_bf16_upstream_gradient_keeps_its_digits(cuda, upstream):
    """Gradients that were stored under 1 are off by one rounding to bf16 (2^-8) after the multiplication, not by the
    rounding of the upstream value too."""
    h, w, labels, b = make(150, 96, 333, torch.bfloat16, True)
    one = backward(h, w, labels, b, "mean", 1.0)
    scaled = backward(h, w, labels, b, "mean", upstream)
    c = float(torch.tensor(upstream))
    for x, y in zip(one[1:], scaled[1:]):
        want = x.double() * c
        rounding = 2.0**-24 if y.dtype == torch.float32 else 2.0**-8
        assert y.dtype == x.dtype and bool(((y.double() - want).abs() <= want.abs() * (rounding + 2.0**-24) + 1e-38).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_backward_under_a_loss_scale_in_a_graph(cuda, dtype):
    from evox_b200.loss_kernels import linear_cross_entropy

    h, w, labels, _ = make(300, 128, 1000, dtype, False)
    hs, ws = h.clone().requires_grad_(), w.clone().requires_grad_()
    scale = torch.tensor(2.0**16, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in torch.autograd.grad(linear_cross_entropy(hs, ws, labels) * scale, (hs, ws))]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(linear_cross_entropy(hs, ws, labels) * scale, (hs, ws))
    for factor in (1.0, 0.25):
        scale.fill_(2.0**16 * factor)
        graph.replay()
        for x, y in zip(want, got):  # a power of two: the same digits
            assert bool(torch.isfinite(y).all())
            if dtype == torch.bfloat16:
                assert torch.equal(x * factor, y)
            else:  # below 2^-14 the scaled gradient has fewer digits
                assert bool(((x.double() * factor - y.double()).abs() <= 2.0**-11 * (x.double() * factor).abs() + 2.0**-24).all())


def test_forward_mode_is_refused():
    """A dual tensor does not require grad; without a look at its tangent the loss would come out as a constant."""
    import torch.autograd.forward_ad as fw

    from evox_b200._cabi import EvoxKernelError
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, y, b = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(9, 16, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64), torch.zeros(9)
    with fw.dual_level():
        for i in (0, 1, 3):
            args = [h, w, y, b]
            args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
            for fn in (linear_cross_entropy, linear_cross_entropy_grad):
                with pytest.raises(EvoxKernelError, match="forward-mode"):
                    fn(*args)
        for fn in (linear_cross_entropy, linear_cross_entropy_grad):  # no tangent: refused for being on the host only
            with pytest.raises(EvoxKernelError, match="CUDA device"):
                fn(h, w, y, b)


@gpu
def test_values_without_a_tangent_pass_inside_a_dual_level(cuda):
    import torch.autograd.forward_ad as fw

    from evox_b200.loss_kernels import linear_cross_entropy

    h, w, labels, b = make(40, 64, 300, torch.bfloat16, True)
    want = linear_cross_entropy(h, w, labels, b)
    with fw.dual_level():
        assert torch.equal(linear_cross_entropy(h, w, labels, b), want)


@gpu
@pytest.mark.parametrize("dtype,reduction", [(torch.bfloat16, "mean"), (torch.bfloat16, "none"), (torch.float16, "sum")])
def test_saved_tensors_are_unpacked_once(cuda, dtype, reduction):
    """Hooks that keep what a graph saves elsewhere (offloading) bring it back once."""
    from evox_b200.loss_kernels import linear_cross_entropy

    h, w, labels, b = make(40, 64, 300, dtype, True)
    hs = h.clone().requires_grad_()
    count = {"pack": 0, "unpack": 0}

    def pack(t):
        count["pack"] += 1
        return t.cpu()

    def unpack(t):
        count["unpack"] += 1
        return t.cuda()

    want, = torch.autograd.grad(linear_cross_entropy(hs, w, labels, b, reduction=reduction).sum(), hs)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        loss = linear_cross_entropy(hs, w, labels, b, reduction=reduction)
    got, = torch.autograd.grad(loss.sum(), hs)
    assert torch.equal(got, want) and count["unpack"] == count["pack"] > 0
