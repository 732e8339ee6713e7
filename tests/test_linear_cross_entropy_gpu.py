"""The vocabulary head's cross entropy and its gradient against the formulas in 64 bits.

Bounds, with u = eps / 2 of the 16-bit type (bf16 2^-8, fp16 2^-11), counted before any run:
  logits     a 32-bit accumulator that may truncate (2^-23 of the running sum per 16 products):
             dz = (hidden / 16 + 8) 2^-23 sum |h w|
  loss       log-sum-exp and the label's logit move by dz each; exponent and logarithm: 2^-21 (max |z| + 16)
  gradients  g = c (p - 1[label]) is rounded twice (exponential, then g): 2 u (1 + u) of c (p + 1[label]); p moves by
             2 dz + 2^-20 (max |z| + 16) of itself; the products truncate as above over their own length; the
             output is rounded once more (u). fp16: subnormal steps of the scaled g (2^-39) and of the output.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
IGNORE = -100
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make(rows, hidden, vocab, dtype, bias, seed=0, ignored=0.2, scale=1.3):
    g = torch.Generator().manual_seed(seed + 7 * rows + 13 * hidden + vocab)
    w = torch.randn(vocab, hidden, generator=g) * (scale / hidden**0.5)
    labels = torch.randint(0, vocab, (rows,), generator=g)
    h = torch.randn(rows, hidden, generator=g) + w[labels] * 3.0
    b = torch.randn(vocab, generator=g) * 0.3 if bias else None
    if rows > 1:
        labels[torch.rand(rows, generator=g) < ignored] = IGNORE
        labels[0], labels[-1] = vocab - 1, 0
    return [None if t is None else t.cuda() for t in (h.to(dtype), w.to(dtype), labels, b)]


class Formula:
    """Values in 64 bits and the bounds above."""

    def __init__(self, h, w, labels, b, reduction="none", g=None):
        dtype, u = h.dtype, U[h.dtype]
        h, w = h.double(), w.double()
        rows, hidden = h.shape
        vocab = w.shape[0]
        z = h @ w.t() + (0 if b is None else b.double())
        valid = labels != IGNORE
        at = torch.where(valid, labels, 0)
        lse = torch.logsumexp(z, dim=1)
        self.loss = torch.where(valid, lse - z.gather(1, at[:, None])[:, 0], 0.0)
        zmax = torch.where(torch.isfinite(z), z.abs(), 0.0).amax(dim=1)
        dz = (hidden / 16 + 8) * 2.0**-23 * ((h.abs() @ w.abs().t()).amax(dim=1) + zmax)
        self.loss_tol = 2 * dz + 2.0**-21 * (zmax + 16)
        count = valid.sum()
        if reduction == "none":
            c = torch.ones(rows, dtype=torch.float64, device=h.device) if g is None else g.double()
        else:
            c = torch.ones(rows, dtype=torch.float64, device=h.device) * (1.0 if g is None else g.double())
            if reduction == "mean":
                c = c / count
            self.loss_tol = (self.loss_tol * valid).sum() / (count if reduction == "mean" else 1) + self.loss.sum().abs() * 2.0**-22 / (
                count if reduction == "mean" else 1)
            self.loss = self.loss.sum() / (count if reduction == "mean" else 1)
        c = torch.where(valid, c, 0.0)[:, None]
        p = torch.exp(z - lse[:, None])
        hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
        G = torch.where(valid[:, None], c * (p - hot), 0.0)
        size = torch.where(valid[:, None], c.abs() * (p + hot), 0.0)
        rel = 2 * u * (1 + u) + 2 * dz[:, None] + 2.0**-20 * (zmax[:, None] + 16) + 2.0**-22
        # (an exponential below 2^-126 becomes 0)
        err = size * rel + (2.0**-38 * c.abs().max() if dtype == torch.float16 else 2.0**-125 * c.abs().max()) * valid[:, None]
        tiny = 2.0**-25 if dtype == torch.float16 else 1e-38
        hv = torch.where(valid[:, None], h, 0.0)
        self.dh, self.dw, self.db = G @ w, G.t() @ hv, G.sum(dim=0)
        self.dh_tol = err @ w.abs() + (vocab / 16 + 8) * 2.0**-23 * (size @ w.abs()) + u * self.dh.abs() + tiny
        self.dw_tol = err.t() @ hv.abs() + (rows / 16 + 8) * 2.0**-23 * (size.t() @ hv.abs()) + u * self.dw.abs() + tiny
        # the bias gradient sums 32-bit values: the exponentials with what their rounding left (off by u u). In fp16 what is
        # left can be subnormal: off by half of the smallest step, 2^-25, of a value that carries 2^15, so 2^-40 of c
        self.db_tol = (size * (rel - 2 * u * (1 + u) + u * u)).sum(dim=0) + (rows + 8) * 2.0**-23 * size.sum(dim=0) + 2.0**-60
        if dtype == torch.float16:
            self.db_tol = self.db_tol + 2.0**-40 * c.abs().sum()


def near(got, want, tol, what):
    got = got.double()
    off = (got - want).abs() - tol
    assert got.shape == want.shape and bool((off <= 0).all()), f"{what}: {float(off.max())} above the bound, largest error {float((got - want).abs().max())}"


SIZES = [(1, 8, 1), (1, 64, 5), (2, 1, 3), (3, 100, 257), (64, 256, 1000), (129, 512, 1009), (255, 72, 128), (256, 64, 256), (257, 1000, 1023),
         (300, 1001, 777), (1024, 256, 4099), (40, 4096, 300), (2000, 136, 70), (65, 64, 300), (128, 200, 1000), (32, 96, 129), (33, 1001, 640),
         (9, 2200, 2500), (1, 4096, 4096),
         (33, 2048, 8000), (64, 1024, 515)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden,vocab", SIZES)
def test_loss(cuda, rows, hidden, vocab, dtype):
    from evox_b200.loss_kernels import linear_cross_entropy

    for bias in (False, True):
        h, w, labels, b = make(rows, hidden, vocab, dtype, bias)
        for reduction in ("none", "sum", "mean"):
            f = Formula(h, w, labels, b, reduction)
            near(linear_cross_entropy(h, w, labels, b, reduction=reduction), f.loss, f.loss_tol, reduction)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden,vocab", SIZES)
def test_gradient(cuda, rows, hidden, vocab, dtype):
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    for bias, reduction, chunk in ((False, "mean", None), (True, "sum", None), (True, "mean", max(1, rows // 3))):
        h, w, labels, b = make(rows, hidden, vocab, dtype, bias)
        f = Formula(h, w, labels, b, reduction)
        loss, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, reduction=reduction, chunk_rows=chunk)
        assert dh.dtype == dw.dtype == dtype
        near(loss, f.loss, f.loss_tol, "loss")
        near(dh, f.dh, f.dh_tol, "dh")
        near(dw, f.dw, f.dw_tol, "dw")
        if bias:
            near(db, f.db, f.db_tol, "db")
        else:
            assert db is None


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_upstream_gradients(cuda, dtype):
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    h, w, labels, b = make(200, 128, 500, dtype, True)
    gen = torch.Generator().manual_seed(1)
    for g in (torch.randn(200, generator=gen).cuda(), torch.rand(200, generator=gen).cuda() * 1e-6, torch.zeros(200, device=cuda)):
        f = Formula(h, w, labels, b, "none", g)
        loss, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, reduction="none", grad_loss=g, chunk_rows=77)
        near(loss, f.loss, f.loss_tol, "loss")
        near(dh, f.dh, f.dh_tol, "dh")
        near(dw, f.dw, f.dw_tol, "dw")
        near(db, f.db, f.db_tol, "db")
    g = torch.tensor(0.37, device=cuda)
    f = Formula(h, w, labels, b, "mean", g)
    _, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, reduction="mean", grad_loss=g)
    near(dh, f.dh, f.dh_tol, "dh")
    near(dw, f.dw, f.dw_tol, "dw")


@gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_autograd_matches_the_formula(cuda, reduction):
    from evox_b200.loss_kernels import linear_cross_entropy

    h, w, labels, b = make(150, 96, 333, torch.bfloat16, True)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    three = leaves[0].view(5, 30, 96)
    loss = linear_cross_entropy(three, leaves[1], labels.view(5, 30), leaves[2], reduction=reduction, chunk_rows=70)
    g = torch.randn(150, generator=torch.Generator().manual_seed(3)).cuda() if reduction == "none" else torch.tensor(1.5, device=cuda)
    loss.backward(g.view(loss.shape))
    f = Formula(h, w, labels, b, reduction, g)
    extra = 1 if reduction == "none" else 2  # a scalar loss scales stored gradients: one rounding more
    near(leaves[0].grad, f.dh, f.dh_tol + (extra - 1) * 2.0**-8 * 1.01 * f.dh.abs(), "dh")
    near(leaves[1].grad, f.dw, f.dw_tol + (extra - 1) * 2.0**-8 * 1.01 * f.dw.abs(), "dw")
    near(leaves[2].grad, f.db, f.db_tol + 2.0**-22 * f.db.abs(), "db")
    only = w.clone().requires_grad_()
    linear_cross_entropy(h, only, labels, b, reduction="sum").backward()
    assert only.grad is not None and torch.isfinite(only.grad).all()


@gpu
def test_gradient_against_differences(cuda):
    """Inputs on a grid of 1 / 16 whose neighbours are exact in bf16: (f(x + d) - f(x - d)) / 2 against grad . d. With
    t = max |change of a logit| along d, the third derivative of log-sum-exp along d is at most (2 t)^3 a row."""
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    g = torch.Generator().manual_seed(0)
    rows, hidden, vocab = 70, 48, 90
    h = (torch.randint(-40, 40, (rows, hidden), generator=g) / 16.0).cuda()
    w = (torch.randint(-6, 6, (vocab, hidden), generator=g) / 16.0).cuda()
    labels = torch.randint(0, vocab, (rows,), generator=g).cuda()
    dir_h = (torch.randint(-1, 2, (rows, hidden), generator=g) * (torch.rand(rows, hidden, generator=g) < 0.1) / 16.0).cuda()
    dir_w = (torch.randint(-1, 2, (vocab, hidden), generator=g) * (torch.rand(vocab, hidden, generator=g) < 0.02) / 16.0).cuda()
    bf = torch.bfloat16

    def f(hh, ww):
        assert torch.equal(hh.to(bf).float(), hh) and torch.equal(ww.to(bf).float(), ww)
        return linear_cross_entropy(hh.to(bf), ww.to(bf), labels, reduction="none").double()

    _, dh, dw, _ = linear_cross_entropy_grad(h.to(bf), w.to(bf), labels, reduction="sum")
    F64 = Formula(h.to(bf), w.to(bf), labels, None, "sum")
    for d_h, d_w, grad, tol, d in ((dir_h, 0 * dir_w, dh, F64.dh_tol, dir_h), (0 * dir_h, dir_w, dw, F64.dw_tol, dir_w)):
        slope = float((f(h + d_h, w + d_w) - f(h - d_h, w - d_w)).sum()) / 2
        t = (d_h @ w.t() + h @ d_w.t()).abs().amax(dim=1).double()
        bound = float(((2 * t) ** 3 / 6).sum()) + float((tol * d.abs()).sum()) + rows * float(Formula(h.to(bf), w.to(bf), labels, None).loss_tol.max())
        assert abs(slope - float((grad.double() * d).sum())) <= bound


@gpu
def test_ignored_rows_may_hold_anything(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, b = make(140, 64, 300, torch.bfloat16, True)
    clean = linear_cross_entropy_grad(h, w, labels, b)
    dirty = h.clone()
    bad = (labels == IGNORE).nonzero()[:, 0]
    assert bad.numel() >= 3
    dirty[bad[0]], dirty[bad[1]], dirty[bad[2]] = float("nan"), float("inf"), torch.finfo(torch.bfloat16).min
    got = linear_cross_entropy_grad(dirty, w, labels, b)
    for x, y in zip(clean, got):
        assert torch.equal(x, y)
    assert torch.equal(linear_cross_entropy(dirty, w, labels, b, reduction="none"), linear_cross_entropy(h, w, labels, b, reduction="none"))
    assert bool((got[1][labels == IGNORE] == 0).all())


@gpu
def test_nothing_but_ignored_rows(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, b = make(9, 64, 300, torch.bfloat16, True)
    labels = torch.full_like(labels, IGNORE)
    assert torch.isnan(linear_cross_entropy(h, w, labels, b))  # 0 / 0, as torch has it
    assert float(linear_cross_entropy(h, w, labels, b, reduction="sum")) == 0.0
    for reduction in ("mean", "sum", "none"):
        _, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, reduction=reduction)
        assert not dh.any() and not dw.any() and not db.any()


@gpu
def test_masked_vocabulary(cuda):
    """Bias entries of -inf or the type's lowest value take words out; a row that keeps one word has loss 0 on it."""
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, _ = make(33, 64, 700, torch.bfloat16, False, ignored=0.0)
    labels[:] = torch.randint(0, 100, (33,), generator=torch.Generator().manual_seed(0)).cuda()
    for low in (float("-inf"), torch.finfo(torch.float32).min):
        b = torch.zeros(700, device=cuda)
        b[100:] = low  # whole 128-column slices hold nothing
        f = Formula(h, w[:100], labels, None, "sum")
        loss, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, reduction="sum")
        near(loss, f.loss, f.loss_tol, "loss")
        near(dh, f.dh, f.dh_tol * 1.01, "dh")
        near(dw[:100], f.dw, f.dw_tol, "dw")
        assert not dw[100:].any() and not db[100:].any()
    b = torch.full((700,), float("-inf"), device=cuda)
    b[3] = 0.0
    labels[:] = 3
    assert float(linear_cross_entropy(h, w, labels, b, reduction="sum")) == 0.0
    labels[:] = 4
    assert bool(torch.isinf(linear_cross_entropy(h, w, labels, b, reduction="none")).all())
    b[3] = float("-inf")  # nothing left: 0 / 0
    assert bool(torch.isnan(linear_cross_entropy(h, w, labels, b, reduction="none")).all())
    # a finite mask over everything leaves 700 equal logits in 32 bits
    b = torch.full((700,), torch.finfo(torch.float32).min, device=cuda)
    equal = torch.full((33,), math.log(700.0), dtype=torch.float64, device=cuda)
    near(linear_cross_entropy(h, w, labels, b, reduction="none"), equal, equal * 2.0**-20, "loss")
    _, dh, _, db = linear_cross_entropy_grad(h, w, labels, b, reduction="sum")
    hot = torch.zeros(700, dtype=torch.float64, device=cuda)
    hot[4] = 33.0
    near(db, 33.0 / 700 - hot, 33.0 / 700 * 2.0**-7 + hot * 2.0**-7, "db")
    assert bool(torch.isfinite(dh).all())


@gpu
def test_labels_outside_the_vocabulary_give_nan(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, _ = make(20, 64, 300, torch.bfloat16, False, ignored=0.0)
    want = linear_cross_entropy(h, w, labels, reduction="none")
    for bad in (300, 383, 511, -1, 2**40, -(2**40)):
        broken = labels.clone()
        broken[7] = bad
        got = linear_cross_entropy(h, w, broken, reduction="none")
        assert torch.isnan(got[7]) and torch.equal(got[:7], want[:7]) and torch.equal(got[8:], want[8:])
        loss, dh, _, _ = linear_cross_entropy_grad(h, w, broken)
        assert torch.isnan(loss) and bool(torch.isnan(dh[7]).all()) and bool(torch.isfinite(dh[:7]).all())


@gpu
def test_infinite_inputs_behave_as_the_formula(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy

    h, w, labels, _ = make(20, 64, 300, torch.bfloat16, False, ignored=0.0)
    h[3, 5] = float("inf")
    h[4, 5] = float("nan")
    got = linear_cross_entropy(h, w, labels, reduction="none")
    assert torch.isnan(got[3]) and torch.isnan(got[4]) and int(torch.isfinite(got).sum()) == 18


@gpu
def test_strides_and_offsets(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    h, w, labels, b = make(100, 64, 300, torch.bfloat16, True)
    want = linear_cross_entropy_grad(h, w, labels, b)
    wide_h, wide_w = torch.full((100, 96), 7.0, dtype=h.dtype, device=cuda), torch.full((300, 72), 7.0, dtype=h.dtype, device=cuda)
    views = []
    wide_h[:, 16:80], wide_w[:, 8:] = h, w
    views.append((wide_h[:, 16:80], wide_w[:, 8:]))            # rows on 16-byte boundaries: used as they are
    odd_h, odd_w = torch.full((100, 67), 7.0, dtype=h.dtype, device=cuda), torch.full((300, 65), 7.0, dtype=h.dtype, device=cuda)
    odd_h[:, 3:], odd_w[:, :64] = h, w
    views.append((odd_h[:, 3:], odd_w[:, :64]))                # not on them: copied
    views.append((h.t().contiguous().t(), w.t().contiguous().t()))
    flat = torch.zeros(100 * 64 + 1, dtype=h.dtype, device=cuda)
    flat[1:] = h.reshape(-1)
    views.append((flat[1:].view(100, 64), w))                  # contiguous, but starting off a boundary
    two = torch.stack([labels, labels], dim=1)[:, 0]
    for hv, wv in views:
        for x, y in zip(want, linear_cross_entropy_grad(hv, wv, two, b)):
            assert torch.equal(x, y)
    row = h[:1].expand(40, 64)                                 # a broadcast row (stride 0)
    same = linear_cross_entropy_grad(row, w, labels[:1].expand(40), b, reduction="none")
    alone = linear_cross_entropy_grad(row.contiguous(), w, labels[:1].expand(40).contiguous(), b, reduction="none")
    for x, y in zip(same, alone):
        assert torch.equal(x, y)


@gpu
def test_no_rows(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    _, w, _, b = make(2, 64, 300, torch.bfloat16, True)
    h, labels = torch.empty(0, 64, dtype=w.dtype, device=cuda), torch.empty(0, dtype=torch.int64, device=cuda)
    assert linear_cross_entropy(h, w, labels, b, reduction="none").shape == (0,)
    assert float(linear_cross_entropy(h, w, labels, b, reduction="sum")) == 0.0 and torch.isnan(linear_cross_entropy(h, w, labels, b))
    _, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b)
    assert dh.shape == (0, 64) and not dw.any() and not db.any()


@gpu
def test_repeats_bit_for_bit_on_other_streams_and_in_graphs(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, labels, b = make(500, 256, 3001, torch.bfloat16, True)
    want = linear_cross_entropy_grad(h, w, labels, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = linear_cross_entropy_grad(h, w, labels, b)
    again = linear_cross_entropy_grad(h, w, labels, b)
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(want, other, again):
        assert torch.equal(x, y) and torch.equal(x, z)
    # two graphs, replayed one after the other and side by side, on inputs that change between replays
    inputs = [t.clone() for t in (h, w, labels)]
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(linear_cross_entropy_grad(*inputs, b) + (linear_cross_entropy(*inputs, b, reduction="none"),))
        graphs.append(graph)
    per_row = linear_cross_entropy(h, w, labels, b, reduction="none")
    for _ in range(2):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.current_stream().wait_stream(side)
        for out in outs:
            for x, y in zip(want + (per_row,), out):
                assert torch.equal(x, y)
    h2, _, labels2, _ = make(500, 256, 3001, torch.bfloat16, True, seed=5)
    inputs[0].copy_(h2)
    inputs[2].copy_(labels2)
    graphs[0].replay()
    for x, y in zip(linear_cross_entropy_grad(h2, w, labels2, b), outs[0]):
        assert torch.equal(x, y)


@gpu
def test_backward_in_a_graph(cuda):
    from evox_b200.loss_kernels import linear_cross_entropy

    h, w, labels, _ = make(300, 128, 1000, torch.bfloat16, False)
    hs, ws = h.clone().requires_grad_(), w.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = torch.autograd.grad(linear_cross_entropy(hs, ws, labels), (hs, ws))
    torch.cuda.current_stream().wait_stream(side)
    want = [t.clone() for t in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(linear_cross_entropy(hs, ws, labels), (hs, ws))
    graph.replay()
    for x, y in zip(want, got):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("rows", [16, 130])
def test_offsets_beyond_32_bits(cuda, rows):
    """A weight of more than 2^31 elements; words on both sides of that are checked in 64 bits, the normaliser comes from
    32-bit products of every word (their error, about 2^-24 sqrt(4096) of a logit near 1, is far below the bounds used)."""
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    hidden, vocab = 4096, 530_001
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(vocab, hidden, dtype=torch.bfloat16, device=cuda).normal_(0.0, 1 / 64, generator=g)
    h = torch.randn(rows, hidden, generator=g, device=cuda).bfloat16()
    labels = torch.randint(0, vocab, (rows,), generator=g, device=cuda)
    labels[0], labels[1] = vocab - 1, 524_289
    loss, dh, dw, _ = linear_cross_entropy_grad(h, w, labels, reduction="none")
    parts = [torch.logsumexp((h.float() @ w[i : i + 65536].float().t()).double(), dim=1) for i in range(0, vocab, 65536)]
    lse = torch.logsumexp(torch.stack(parts), dim=0)
    want = lse - (h.double() * w[labels].double()).sum(dim=1)
    assert float((loss.double() - want).abs().max()) <= 1e-4
    words = torch.cat([torch.tensor([0, 524_287, 524_288, 524_289, vocab - 2, vocab - 1], device=cuda), labels])
    p = torch.exp(h.double() @ w[words].double().t() - lse[:, None]) - (labels[:, None] == words[None, :]).double()
    near(dw[words], p.t() @ h.double(), (p.abs().t() @ h.double().abs()) * 2.0**-6 + 1e-30, "dw")
    del dw
    back = -w[labels].double()
    for i in range(0, vocab, 65536):
        piece = w[i : i + 65536].float()
        back += (torch.exp((h.float() @ piece.t()) - lse[:, None].float()) @ piece).double()
    size = torch.exp(h.float() @ w[:65536].float().t() - lse[:, None].float()) @ w[:65536].float().abs() * (vocab / 65536 * 1.5) + w[labels].abs().float()
    near(dh, back, size.double() * 2.0**-6, "dh")


@gpu
def test_no_wait_expired_and_a_status_is_reported_once(cuda):
    from evox_b200._cabi import EvoxKernelError
    from evox_b200.lora_kernels import raise_on_kernel_errors, status_word

    raise_on_kernel_errors()
    assert status_word(cuda) is status_word(torch.device("cuda:0"))
    status_word(cuda).fill_(4)  # what a kernel whose wait expired would leave
    with pytest.raises(EvoxKernelError, match="status 4"):
        raise_on_kernel_errors()
    raise_on_kernel_errors()


# ---- refusals: host checks, no device needed ------------------------------------------------------------------


def test_refusals():
    from evox_b200._cabi import EvoxKernelError
    from evox_b200.loss_kernels import linear_cross_entropy, linear_cross_entropy_grad

    h, w, y = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(9, 16, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for args, kw, said in (((h, w, y), {}, "CUDA device"), ((h.float(), w.float(), y), {}, "bfloat16"), ((h, w.half(), y), {}, "bfloat16"),
                           ((h, w[:, :8], y), {}, "shape mismatch"), ((h, w[:0], y), {}, "shape mismatch"), ((h, w, y.int()), {}, "int64"),
                           ((h, w, y[:3]), {}, "labels"), ((h, w, y, torch.zeros(8)), {}, "bias"), ((h, w, y), {"reduction": "max"}, "reduction"), ((h, w, y), {"chunk_rows": 0}, "chunk_rows")):
        for fn in (linear_cross_entropy, linear_cross_entropy_grad):
            with pytest.raises(EvoxKernelError, match=said):
                fn(*args, **kw)


def test_c_entry_refuses_bad_arguments():
    from evox_b200 import _cabi

    lib = _cabi.lib
    good = dict(h=256, ld_h=64, w=256, ld_w=64, dtype=0, bias=None, labels=256, ignore=-100, rows=4, hidden=64, vocab=9, reduction=0, loss=256,
                ws=256, nbytes=1 << 20, err=256, stream=None)  # never launched: every call below is refused first

    def call(**kw):
        return lib.evox_linear_cross_entropy(*{**good, **kw}.values())

    for kw in (dict(h=None), dict(labels=None), dict(loss=None), dict(ws=None), dict(err=None), dict(rows=0), dict(rows=-1), dict(hidden=0),
               dict(vocab=0), dict(vocab=1 << 40), dict(rows=1 << 29, vocab=1 << 25), dict(dtype=2), dict(reduction=3), dict(ld_h=60), dict(ld_w=56), dict(h=257), dict(w=259),
               dict(ws=128)):
        assert call(**kw) == -1, kw
        assert b"linear_cross_entropy" in lib.evox_last_error()
    assert call(nbytes=16) == -3
    assert lib.evox_linear_cross_entropy_workspace_bytes(0, 4, 4, 0) == 0
    assert [lib.evox_linear_cross_entropy_copies(*a) for a in ((256, 64, 256, 64), (258, 64, 256, 64), (256, 64, 256, 65), (264, 8, 272, 12))] == [0, 1, 2, 3]
    plain = lib.evox_linear_cross_entropy_workspace_bytes(4, 63, 9, 0)
    assert lib.evox_linear_cross_entropy_workspace_bytes(4, 63, 9, 1) == plain + 512 and lib.evox_linear_cross_entropy_workspace_bytes(4, 63, 9, 2) == plain + 1280
    rows, vocab = 100000, 131072
    assert lib.evox_linear_cross_entropy_chunk_rows(rows, vocab) == 8192 and lib.evox_linear_cross_entropy_chunk_rows(100, vocab) == 100
    small = lib.evox_linear_cross_entropy_grad_workspace_bytes(rows, 64, vocab, 256, 0, 0)
    assert small < lib.evox_linear_cross_entropy_grad_workspace_bytes(rows, 64, vocab, 512, 0, 0)
