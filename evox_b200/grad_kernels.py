"""Global gradient norm over many tensors, and clipping by it, on the CUDA kernels."""

from __future__ import annotations

from array import array
from collections.abc import Iterable
from operator import attrgetter

import torch

from . import _cabi

__all__ = ["grad_norm", "clip_grad_norm_"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _norm(tensors: torch.Tensor | Iterable[torch.Tensor], max_norm: float, clip: bool) -> torch.Tensor:
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    err = _cabi.EvoxKernelError
    n = len(tensors)
    if n == 0:
        raise err("the list of gradients is empty")
    # whole-list passes instead of a loop with several calls per tensor: a list of hundreds costs tens of microseconds
    types = set(map(attrgetter("dtype"), tensors))
    devices = set(map(torch.Tensor.get_device, tensors))
    if not types <= _DTYPES.keys():
        raise err(f"gradients must be bfloat16, float16 or float32, got {sorted(map(str, types - _DTYPES.keys()))}")
    if len(devices) != 1 or -1 in devices:
        raise err(f"gradients must live on one CUDA device (evox_b200 has no CPU path), got {sorted({str(t.device) for t in tensors})}")
    if devices != {torch.cuda.current_device()}:
        _cabi.ptr(tensors[0][:0] if tensors[0].ndim else tensors[0], None, "gradients")  # names both devices
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        raise err("gradients must be contiguous")
    dev = tensors[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = _cabi.lib.evox_grad_norm_workspace_bytes(n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    table = (array("Q", map(torch.Tensor.data_ptr, tensors)), array("q", map(torch.Tensor.numel, tensors)),
             array("i", [_DTYPES[types.pop()]]) * n if len(types) == 1 else array("i", [_DTYPES[t.dtype] for t in tensors]))
    _cabi.check(_cabi.lib.evox_clip_grad_norm(*(a.buffer_info()[0] for a in table), n, max_norm, int(clip), norm.data_ptr(), ws.data_ptr(),
                                              nbytes, _cabi.stream_ptr(dev)))
    return norm


def grad_norm(tensors: torch.Tensor | Iterable[torch.Tensor]) -> torch.Tensor:
    """2-norm over all elements of the gradients (contiguous bf16, fp16 or fp32 tensors, mixed types
    allowed): a 0-d fp32 tensor. Sums are made in 64 bits in a fixed order."""
    return _norm(tensors, 0.0, False)


def clip_grad_norm_(tensors: torch.Tensor | Iterable[torch.Tensor], max_norm: float) -> torch.Tensor:
    """Scale the gradients in place by min(1, max_norm / (norm + 1e-6)) and return the norm they had, as
    `torch.nn.utils.clip_grad_norm_` does with its parameters' gradients. Takes the gradients themselves; no two may
    share memory. Nothing is read back: a norm that is not finite turns the gradients into zeros (inf) or NaN, and shows
    in the returned tensor."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _cabi.EvoxKernelError(f"max_norm must not be negative or NaN, got {max_norm}")
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    norm = _norm(tensors, max_norm, True)
    torch.autograd.graph.increment_version(tensors)
    return norm
