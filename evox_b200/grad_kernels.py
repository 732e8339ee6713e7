"""Global gradient norm over many tensors, and clipping by it, on the CUDA kernels."""

from __future__ import annotations

from collections.abc import Iterable
from ctypes import c_int32, c_int64, c_uint64
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
    types = list(map(attrgetter("dtype"), tensors))
    devices = set(map(torch.Tensor.get_device, tensors))
    if not set(types) <= _DTYPES.keys():
        raise err(f"gradients must be bfloat16, float16 or float32, got {sorted(map(str, set(types) - _DTYPES.keys()))}")
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
    _cabi.check(_cabi.lib.evox_clip_grad_norm(
        (c_uint64 * n)(*map(torch.Tensor.data_ptr, tensors)), (c_int64 * n)(*map(torch.Tensor.numel, tensors)),
        (c_int32 * n)(*map(_DTYPES.__getitem__, types)), n, max_norm, int(clip), norm.data_ptr(), ws.data_ptr(), nbytes,
        _cabi.stream_ptr(dev)))
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
