"""Sizes at the ends of what the vocabulary head's cross entropy accepts."""
import pytest
import torch

from tests.test_linear_cross_entropy_gpu import make, near

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("rows,bias", [(3, False), (40, True)])
def test_more_features_than_a_32_bit_product_of_blocks_and_chunks(cuda, rows, bias):
    """12.1 million features: 189,063 blocks of the reduction in 11,817 chunks. With S the largest partial sum of a logit:
    the four accumulators of a chunk truncate 16 times each (2^-23 of what they hold, together at most sum |h w|), and are
    joined with four roundings a chunk (2^-24 S). The softmax moves by twice that; the rest as for other sizes: g
    is rounded twice and the output once (u each)."""
    from evox_b200.loss_kernels import linear_cross_entropy_grad

    hidden, vocab, u = 12_100_000, 5, 2.0**-8
    h, w, labels, b = make(rows, hidden, vocab, torch.bfloat16, bias)
    loss, dh, dw, db = linear_cross_entropy_grad(h, w, labels, b, reduction="sum")
    z = torch.zeros(rows, vocab, dtype=torch.float64, device=cuda)
    absolute, partial = torch.zeros_like(z), torch.zeros_like(z)
    for at in range(0, hidden, 2**16):
        hp, wp = h[:, at : at + 2**16].double(), w[:, at : at + 2**16].double()
        z += hp @ wp.t()
        absolute += hp.abs() @ wp.abs().t()
        partial = torch.maximum(partial, z.abs() + 2**8 * hp.abs().amax() * wp.abs().amax())
    dz = (16 * 2.0**-23 * absolute + 4 * 11_817 * 2.0**-24 * partial).amax(dim=1)
    z += 0.0 if b is None else b.double()
    valid = labels != -100
    at = torch.where(valid, labels, 0)
    lse = torch.logsumexp(z, dim=1)
    want = torch.where(valid, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    slack = 2 * dz + 2.0**-21 * (z.abs().amax(dim=1) + 16)
    near(loss, want.sum(), (slack * valid).sum() + 2.0**-22 * want.sum(), "loss")
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    grad, size = torch.where(valid[:, None], p - hot, 0.0), torch.where(valid[:, None], p + hot, 0.0)
    moved = torch.expm1(2 * dz)[:, None] * p + (2 * u * (1 + u) + 2.0**-19) * size
    moved = torch.where(valid[:, None], moved, 0.0)
    for at in range(0, hidden, 2**20):
        hp, wp = h[:, at : at + 2**20].double(), w[:, at : at + 2**20].double()
        a = grad @ wp
        near(dh[:, at : at + 2**20], a, moved @ wp.abs() + (u + 2.0**-19) * a.abs() + 2.0**-19 * (size @ wp.abs()) + 1e-30, "dh")
        a = grad.t() @ hp
        near(dw[:, at : at + 2**20], a, moved.t() @ hp.abs() + (u + 2.0**-19) * a.abs() + 2.0**-19 * (size.t() @ hp.abs()) + 1e-30, "dw")
    if bias:
        near(db, grad.sum(dim=0), moved.sum(dim=0), "db")


def test_the_largest_vocabulary_of_a_gradient():
    """One word more than the rescaling pass has blocks for is refused before anything is launched (the addresses are made up)."""
    from evox_b200 import _cabi

    lib = _cabi.lib
    good = dict(h=256, ld_h=8, w=256, ld_w=8, dtype=0, bias=None, labels=256, ignore=-100, rows=4, hidden=8, vocab=67_105_793, reduction=0, grad_loss=None,
                chunk=4, loss=256, dh=256, dw=256, db=None, ws=256, nbytes=0, err=256, stream=None)
    assert lib.evox_linear_cross_entropy_grad(*good.values()) == -1
    assert b"vocab must be at most 67105792" in lib.evox_last_error()
    assert lib.evox_linear_cross_entropy_grad(*{**good, "vocab": 67_105_792}.values()) == -3  # this one has no workspace
