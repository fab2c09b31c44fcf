"""The global norm of a list of gradients, and clipping by it, on the GPU.

What the reference's training loop does between its backward pass and the optimizer (train/runners.py:378-380,
``torch.nn.utils.clip_grad_norm_``): the 2-norm over all gradients, and all of them times ``min(1, max_norm / (norm + 1e-6))``.
``lbi_clip_gradients`` takes the whole list in two launches per 140 tensors, whatever their sizes and types, and the
norm stays on the device.
"""
from __future__ import annotations

import array
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


def _refuse(tensors: Sequence[torch.Tensor], what: str, index: int) -> None:
    """Raises for the first of ``tensors`` that the kernels do not take on the device ``index``."""
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} must be torch.Tensors")
        if t.layout != torch.strided:
            raise TypeError(f"{what} must be dense tensors")
        _lib.dtype_code(t.dtype)
        if not t.is_cuda:
            raise RuntimeError(f"{what} must be CUDA tensors (this build has no CPU execution path)")
        if t.get_device() != index:
            raise ValueError(f"{what} must be on one device")


def _clip(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor] | None, max_norm: float) -> torch.Tensor:
    """``outs``: where the results go (``grads`` itself: in place; ``None``: nowhere, the norm alone)."""
    if not isinstance(grads[0], torch.Tensor) or not grads[0].is_cuda:
        _refuse(grads[:1], "grads", 0)
    index, codes, changing = grads[0].get_device(), _lib._DTYPE_CODES, torch.is_grad_enabled()
    words, held, late = [], [], []
    for i, g in enumerate(grads):
        out = None if outs is None else outs[i]
        try:  # most calls: a tensor costs less than a microsecond
            dtype = g.dtype
            if out is not None and out is not g:
                if g.shape != out.shape or out.dtype is not dtype:
                    raise ValueError("out must have the shapes and types of the gradients")
                plain = g.is_contiguous() and out.is_contiguous() and out.get_device() == index
            else:
                plain = g.is_contiguous()
            if plain and g.get_device() == index and not (changing and out is not None and out.requires_grad):
                words += (g.data_ptr(), 0 if out is None else out.data_ptr(), g.numel(), codes[dtype])
                continue
        except (AttributeError, KeyError, RuntimeError):
            pass  # said below
        _refuse([g], "grads", index)
        to = out
        if out is not None:
            _refuse([out], "out", index)
            if out.requires_grad and changing:
                raise RuntimeError("clip_gradients writes tensors that require grad: call it under torch.no_grad()")
        if not _flat(g) or not (out is None or out is g or out.stride() == g.stride()):
            g = g.contiguous()
            if out is not None and (out is grads[i] or not out.is_contiguous()):
                to = torch.empty_like(g)
                late.append((out, to))
            # a contiguous `out` of its own is written by the kernel
            held.append((g, to))  # copies live until the kernels are queued
        words += (g.data_ptr(), 0 if to is None else to.data_ptr(), g.numel(), codes[g.dtype])
    if late and len({(o.data_ptr(), o.shape, o.stride()) for o, _ in late}) != len(late):
        raise ValueError("a result overlaps another tensor")
    count, device = len(grads), grads[0].device
    table = array.array("q", words)  # lbi_gradient of include/lbi_hip.h: four words of 64 bits
    norm = torch.empty((), device=device, dtype=torch.float32)
    lib = _lib.load()
    with _lib.device_guard(device):
        need = lib.lbi_clip_gradients_workspace_bytes(count)
        workspace = torch.empty(need, device=device, dtype=torch.uint8)
        status = lib.lbi_clip_gradients(table.buffer_info()[0], count, max_norm, norm.data_ptr(), workspace.data_ptr(), need, _lib.current_stream_ptr(device))
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
    return _clip(grads, None, math.inf)


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
    return _clip(grads, grads if out is None else out, max_norm)


__all__ = ["clip_gradients", "gradient_norm"]
