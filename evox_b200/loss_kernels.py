"""Softmax cross entropy of a linear vocabulary head, without its logits, on the tensor cores.

`linear_cross_entropy` is `F.cross_entropy(F.linear(h, weight, bias), labels)` for 16-bit operands: the product's
epilogue reduces every row to its log-sum-exp, so the (rows, vocab) logits never exist. It is differentiable;
`linear_cross_entropy_grad` returns loss and gradients in one call, without autograd. The same loss for a
virtual-LoRA population is `lora_kernels.lora_layer_cross_entropy`.

Every device-side wait is bounded. If one expires, that call and those after it on the device give NaN, losses and
gradients alike, until `lora_kernels.raise_on_kernel_errors` has raised it (a wait for the current stream; once per epoch or
wherever a loss is looked at is enough).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _cabi
from .lora_kernels import status_word

__all__ = ["linear_cross_entropy", "linear_cross_entropy_grad"]

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _operand(x: torch.Tensor, rows: int, hidden: int) -> tuple[torch.Tensor, int, bool]:
    """`x` (rows, hidden) with dense rows, its row stride, and whether its rows start off 16-byte boundaries (the kernels
    then copy it to their workspace)."""
    stride, step = x.stride()
    if rows == 1:
        stride = (hidden + 7) // 8 * 8
    if (step != 1 and hidden != 1) or stride < hidden:
        x, stride = x.detach().contiguous(), hidden
    return x, stride, stride % 8 != 0 or x.data_ptr() % 16 != 0


def _refuse(h, weight, labels, bias, reduction):
    """Say what is wrong with the arguments."""
    err = _cabi.EvoxKernelError
    if reduction not in _REDUCTIONS:
        raise err(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if h.dtype not in _DTYPES or weight.dtype != h.dtype:
        raise err(f"hidden states and weight must both be bfloat16 or both float16, got {h.dtype} and {weight.dtype}")
    if weight.ndim != 2 or h.ndim < 1 or h.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise err(f"shape mismatch: hidden states {tuple(h.shape)}, weight {tuple(weight.shape)}")
    if labels.dtype != torch.int64 or labels.shape != h.shape[:-1]:
        raise err(f"labels must be int64 of shape {tuple(h.shape[:-1])}, got {labels.dtype} {tuple(labels.shape)}")
    if bias is not None and (bias.shape != weight.shape[:1] or not bias.is_floating_point()):
        raise err(f"bias must be floating point of shape ({weight.shape[0]},), got {bias.dtype} {tuple(bias.shape)}")
    for name, t in (("hidden states", h), ("weight", weight), ("labels", labels), ("bias", bias)):
        if t is not None:
            _cabi.ptr(t.reshape(-1)[:0], None, name)  # on a CUDA device, and on the current one


def _arguments(h, weight, labels, bias, reduction):
    """Checked and flattened arguments: (h, weight, labels, bias fp32, leading shape)."""
    dtype, shape = h.dtype, h.shape
    rest = shape[:-1]
    here = torch.cuda.current_device() if h.is_cuda else -1
    if (dtype not in _DTYPES or weight.dtype != dtype or weight.ndim != 2 or not shape or weight.shape[1] != shape[-1] or weight.numel() == 0
            or reduction not in _REDUCTIONS or labels.dtype != torch.int64 or labels.shape != rest
            or h.get_device() != here or weight.get_device() != here or labels.get_device() != here or here < 0
            or (bias is not None and (bias.shape != weight.shape[:1] or not bias.is_floating_point() or bias.get_device() != here))):
        _refuse(h, weight, labels, bias, reduction)
        raise _cabi.EvoxKernelError("arguments of linear_cross_entropy do not fit together")
    if len(shape) != 2:
        h, labels = h.reshape(-1, shape[-1]), labels.reshape(-1)
    if not labels.is_contiguous():
        labels = labels.contiguous()
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_contiguous()):
        bias = bias.detach().to(torch.float32).contiguous()
    return h, weight, labels, bias, rest


def _refuse_tangents(*tensors) -> None:
    """Forward-mode tangents would be dropped without a word: the kernels see values only."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _cabi.EvoxKernelError("linear_cross_entropy has no forward-mode derivative: an argument carries a tangent")


def _check_chunk(chunk_rows: int | None) -> None:
    if chunk_rows is not None and chunk_rows < 1:
        raise _cabi.EvoxKernelError(f"chunk_rows must be at least 1, got {chunk_rows}")


def _loss(h, weight, labels, bias, ignore_index, reduction, shape):
    dev = h.device
    rows, hidden = h.shape
    vocab = weight.shape[0]
    if rows == 0:
        return torch.full(shape if reduction == "none" else (), float("nan") if reduction == "mean" else 0.0, device=dev)
    (h, ld_h, copy_h), (weight, ld_w, copy_w) = _operand(h, rows, hidden), _operand(weight, vocab, hidden)
    loss = torch.empty(shape if reduction == "none" else (), dtype=torch.float32, device=dev)
    lib = _cabi.lib
    nbytes = lib.evox_linear_cross_entropy_workspace_bytes(rows, hidden, vocab, copy_h + 2 * copy_w)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _cabi.check(lib.evox_linear_cross_entropy(
        h.data_ptr(), ld_h, weight.data_ptr(), ld_w, _DTYPES[h.dtype], None if bias is None else bias.data_ptr(), labels.data_ptr(),
        ignore_index, rows, hidden, vocab, _REDUCTIONS[reduction], loss.data_ptr(), ws.data_ptr(), nbytes, status_word(dev).data_ptr(),
        _cabi.stream_ptr(dev)))
    return loss


def _loss_and_grad(h, weight, labels, bias, ignore_index, reduction, shape, grad_loss, chunk_rows, wanted):
    """(loss, dh (rows, hidden), dw, dbias fp32); `wanted`: which of the three gradients are computed."""
    dev, dtype = h.device, h.dtype
    rows, hidden = h.shape
    vocab = weight.shape[0]
    dh = torch.empty(rows, hidden, dtype=dtype, device=dev) if wanted[0] else None
    dw = torch.empty(vocab, hidden, dtype=dtype, device=dev) if wanted[1] else None
    db = torch.empty(vocab, dtype=torch.float32, device=dev) if wanted[2] and bias is not None else None
    if rows == 0:
        return _loss(h, weight, labels, bias, ignore_index, reduction, shape), dh, *(None if g is None else g.zero_() for g in (dw, db))
    (h, ld_h, copy_h), (weight, ld_w, copy_w) = _operand(h, rows, hidden), _operand(weight, vocab, hidden)
    loss = torch.empty(shape if reduction == "none" else (), dtype=torch.float32, device=dev)
    lib = _cabi.lib
    chunk = lib.evox_linear_cross_entropy_chunk_rows(rows, vocab) if chunk_rows is None else chunk_rows
    nbytes = lib.evox_linear_cross_entropy_grad_workspace_bytes(rows, hidden, vocab, chunk, db is not None, copy_h + 2 * copy_w)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _cabi.check(lib.evox_linear_cross_entropy_grad(
        h.data_ptr(), ld_h, weight.data_ptr(), ld_w, _DTYPES[dtype], None if bias is None else bias.data_ptr(), labels.data_ptr(),
        ignore_index, rows, hidden, vocab, _REDUCTIONS[reduction], None if grad_loss is None else grad_loss.data_ptr(), chunk,
        loss.data_ptr(), None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
        ws.data_ptr(), nbytes, status_word(dev).data_ptr(), _cabi.stream_ptr(dev)))
    return loss, dh, dw, db


def linear_cross_entropy_grad(h: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, bias: torch.Tensor | None = None, *,
                              ignore_index: int = -100, reduction: str = "mean", grad_loss: torch.Tensor | None = None,
                              chunk_rows: int | None = None):
    """Loss and its gradients in one call: `(loss, dh, dweight, dbias)`, the gradients in their operands' types
    (`dbias` is None without a bias). Arguments as for `linear_cross_entropy`; `grad_loss` is the upstream gradient
    (one fp32 value, or one per row with `reduction="none"`). `chunk_rows`: rows whose 16-bit exponentials
    are held at a time (default: all, up to 2 GiB of them; a bias gradient doubles the bytes)."""
    _check_chunk(chunk_rows)
    _refuse_tangents(h, weight, bias, grad_loss)
    flat, weight, labels, bias_f, shape = _arguments(h, weight, labels, bias, reduction)
    if grad_loss is not None:
        want = shape if reduction == "none" else ()
        if grad_loss.shape != want:
            raise _cabi.EvoxKernelError(f"grad_loss must have shape {tuple(want)}, got {tuple(grad_loss.shape)}")
        grad_loss = grad_loss.detach().to(device=flat.device, dtype=torch.float32).contiguous()
    loss, dh, dw, db = _loss_and_grad(flat, weight, labels, bias_f, ignore_index, reduction, shape, grad_loss, chunk_rows, (True, True, True))
    if bias is not None and bias.dtype != torch.float32:
        db = db.to(bias.dtype)
    return loss, dh if dh.shape == h.shape else dh.view(h.shape), dw, db


class _LinearCrossEntropy(torch.autograd.Function):
    """A scalar loss of bf16 operands computes its gradients with the forward pass, while the exponentials are there, and
    backward multiplies them by the upstream gradient (in 32 bits, one more rounding to bf16). Elsewhere backward computes
    them: per-row losses have one upstream value per row, and fp16 would lose what a loss scale is there to keep (numbers
    below 6e-8, or above 65,504 before a small factor) if it rounded before the upstream value is applied."""

    @staticmethod
    def forward(ctx, h, weight, labels, bias, ignore_index, reduction, chunk_rows):
        flat, w, flat_labels, bias_f, shape = _arguments(h, weight, labels, bias, reduction)
        wanted = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3])
        ctx.args = (ignore_index, reduction, shape, h.shape, None if bias is None else bias.dtype, chunk_rows)
        if reduction == "none" or h.dtype == torch.float16:
            ctx.save_for_backward(h, weight, labels, bias)
            return _loss(flat, w, flat_labels, bias_f, ignore_index, reduction, shape)
        loss, *grads = _loss_and_grad(flat, w, flat_labels, bias_f, ignore_index, reduction, shape, None, chunk_rows, wanted)
        ctx.save_for_backward(*grads)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ignore_index, reduction, shape, h_shape, bias_dtype, chunk_rows = ctx.args
        saved = ctx.saved_tensors
        if len(saved) == 4:  # the operands; otherwise gradients
            h, weight, labels, bias = saved
            flat, w, flat_labels, bias_f, _ = _arguments(h, weight, labels, bias, reduction)
            wanted = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3])
            with torch.cuda.device(h.device):
                _, dh, dw, db = _loss_and_grad(flat, w, flat_labels, bias_f, ignore_index, reduction, shape,
                                               grad.to(torch.float32).contiguous(), chunk_rows, wanted)
        else:
            # one element, not a 0-d tensor: that would be rounded to bf16 before the product
            dh, dw, db = (None if g is None else torch.mul(g, grad.reshape(1), out=torch.empty_like(g)) for g in saved)
        return (None if dh is None else dh.view(h_shape), dw, None, None if db is None else db.to(bias_dtype), None, None, None)


def linear_cross_entropy(h: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, bias: torch.Tensor | None = None, *,
                         ignore_index: int = -100, reduction: str = "mean", chunk_rows: int | None = None) -> torch.Tensor:
    """`F.cross_entropy(F.linear(h, weight, bias), labels)` in fp32 without the logits.

    `h` (..., hidden) and `weight` (vocab, hidden): both bf16 or both fp16, any sizes and row strides (rows that do not
    start on 16-byte boundaries are copied); `labels` (...) int64; `bias` (vocab,). Rows labelled `ignore_index`
    have loss 0, do not count in the mean and get zero gradients, whatever they hold; a label
    outside the vocabulary gives NaN. `reduction`: "mean", "sum" or "none" (losses shaped like `labels`).
    Differentiable once in `h`, `weight` and `bias`, in reverse mode (a forward-mode tangent is refused). The softmax gradient
    is rounded to the operands' type before its two products; a mean or sum of bf16 operands stores dh and dweight from the
    forward pass on, elsewhere backward computes them. The gradient holds 16-bit exponentials of `chunk_rows` rows at a time
    (default: all, up to 2 GiB of them; a bias gradient doubles the bytes)."""
    _check_chunk(chunk_rows)
    _refuse_tangents(h, weight, bias)
    if torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearCrossEntropy.apply(h, weight, labels, bias, ignore_index, reduction, chunk_rows)
    return _loss(*_arguments(h, weight, labels, bias, reduction)[:4], ignore_index, reduction, tuple(h.shape[:-1]))
