"""The global norm of a list of gradients, and clipping by it, on the GPU.

What the reference's training loop does between its backward pass and the optimizer (train/runners.py:378-380,
``torch.nn.utils.clip_grad_norm_``): the 2-norm over all gradients, and all of them times ``min(1, max_norm / (norm + 1e-6))``.
``lbi_clip_gradients`` takes the whole list in two launches per hundred tensors, whatever their sizes and types, and the
norm stays on the device.
"""
from __future__ import annotations

import ctypes
import math
from typing import Sequence

import torch

from ... import _lib


def _flat(t: torch.Tensor) -> bool:
    """Whether the elements of ``t`` fill one piece of memory, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda d: t.stride(d), reverse=True)
    return t.permute(order).is_contiguous()


def _check(tensors: Sequence[torch.Tensor], what: str, device: torch.device | None = None) -> torch.device:
    """The one device of ``tensors``."""
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} must be torch.Tensors")
        if t.layout is not torch.strided:
            raise TypeError(f"{what} must be dense tensors")
        if t.dtype not in _lib._DTYPE_CODES:
            _lib.dtype_code(t.dtype)
        if device is None or t.device != device:
            if not t.is_cuda:
                raise RuntimeError(f"{what} must be CUDA tensors (this build has no CPU execution path)")
            if device is not None:
                raise ValueError(f"{what} must be on one device")
            device = t.device
    return device


def _clip(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor | None], max_norm: float) -> torch.Tensor:
    device = grads[0].device
    codes = _lib._DTYPE_CODES
    words, held, late = [], [], []
    for g, out in zip(grads, outs):
        to = out
        if not (g.is_contiguous() and (out is None or out is g or out.is_contiguous())) and not (
                _flat(g) and (out is None or out is g or out.stride() == g.stride())):
            g = g.contiguous()
            if out is not None and (out is g or not out.is_contiguous()):
                to = torch.empty_like(g)
                late.append((out, to))
            # a contiguous `out` of its own is written by the kernel
            held.append((g, to))  # copies live until the kernels are queued
        words += (g.data_ptr(), 0 if to is None else to.data_ptr(), g.numel(), codes[g.dtype])
    count = len(words) // 4
    if late and len({(o.data_ptr(), o.shape, o.stride()) for o, _ in late}) != len(late):
        raise ValueError("a result overlaps another tensor")
    table = (ctypes.c_int64 * len(words))(*words)
    norm = torch.empty((), device=device, dtype=torch.float32)
    lib = _lib.load()
    with _lib.device_guard(device):
        need = int(lib.lbi_clip_gradients_workspace_bytes(table, count))
        workspace = torch.empty(max(need, 8), device=device, dtype=torch.uint8)
        status = lib.lbi_clip_gradients(table, count, max_norm, norm.data_ptr(), workspace.data_ptr(), need,
                                        _lib.current_stream_ptr(device))
    _lib.check(status, "lbi_clip_gradients")
    for out, to in late:
        out.copy_(to)
    return norm


def gradient_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all elements of all ``grads`` (fp32, fp16, bf16, mixed), a scalar tensor of fp32 on their device.
    Squares are added in 64 bits.  An empty list has the norm 0 (on the CPU)."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    _check(grads, "grads")
    return _clip(grads, [None] * len(grads), math.inf)


def clip_gradients(grads: Sequence[torch.Tensor], max_norm: float, *, out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """``out[i] = grads[i] * min(1, max_norm / (norm + 1e-6))``, ``norm`` the 2-norm over all of ``grads``; in place
    without ``out``.  Returns ``norm``, a scalar tensor of fp32 on the device: nothing here waits for it.

    ``out[i]`` has the shape and type of ``grads[i]`` and is ``grads[i]`` itself or overlaps no gradient and no other
    result; the same gradient twice in the list counts twice and needs an ``out`` for each.  As
    ``torch.nn.utils.clip_grad_norm_`` does: a norm that is not a number makes every result one, an infinite norm makes
    finite elements 0.  In place and with a norm below the limit, nothing is written."""
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError("out must hold one tensor for each gradient")
    if not grads:
        return torch.zeros(())
    device = _check(grads, "grads")
    if out is None:
        out = grads
    else:
        _check(out, "out", device)
        for g, o in zip(grads, out):
            if g.shape != o.shape or g.dtype != o.dtype:
                raise ValueError("out must have the shapes and types of the gradients")
    if any(o.requires_grad for o in out) and torch.is_grad_enabled():
        raise RuntimeError("clip_gradients writes tensors that require grad: call it under torch.no_grad()")
    return _clip(grads, out, max_norm)


__all__ = ["clip_gradients", "gradient_norm"]
