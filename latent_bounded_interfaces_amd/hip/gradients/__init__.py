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
from torch.autograd import forward_ad

from ... import _lib


def _flat(t: torch.Tensor) -> bool:
    """Whether the elements of ``t`` fill one piece of memory, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda d: t.stride(d), reverse=True)
    return t.permute(order).is_contiguous()


def _bytes(t: torch.Tensor) -> tuple[int, int]:
    """First byte of ``t`` and the one behind its last."""
    begin, size = t.data_ptr(), t.element_size()
    return begin, begin + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _column(t: torch.Tensor) -> tuple[int, int, int]:
    """``(pitch, begin, end)``: the largest stride in bytes, and where within it all bytes of ``t`` lie, if they do not reach around its end
    (0 for the pitch otherwise, and without a stride)."""
    size = t.element_size()
    dims = [(s * size, n - 1) for s, n in zip(t.stride(), t.shape) if n > 1]
    pitch = max(dims, default=(0, 0))[0]
    if not pitch:
        return 0, 0, 0
    begin = t.data_ptr() % pitch
    end = begin + size + sum(s * most for s, most in dims if s < pitch)
    return (pitch, begin, end) if end <= pitch else (0, 0, 0)


def _solvable(terms: list[tuple[int, int]], target: int, steps: list[int]) -> bool:
    """Whether ``target`` is the sum of ``c * x`` over ``terms`` ``(c, most)``, c descending, each x a whole number of [0, most].  The largest c
    leaves few x whose rest the others can make: strides of a tensor exceed what its inner dimensions span, as a rule.  ``steps`` counts
    down; where they run out the answer is yes."""
    rest = sum(c * most for c, most in terms)
    if not 0 <= target <= rest:
        return False
    if target in (0, rest):
        return True
    (c, most), inner = terms[0], terms[1:]
    rest -= c * most
    for x in range(min(most, target // c), max(0, -((rest - target) // c)) - 1, -1):
        steps[0] -= 1
        if steps[0] < 0 or _solvable(inner, target - c * x, steps):
            return True
    return False


_STEPS = 20_000  # of a search, some 10 ms


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether elements of ``a`` and ``b`` share a byte: a's address + strides * x + byte = b's likewise, b's indexes counted from the end."""
    most: dict[int, int] = {}
    for t in (a, b):
        for c, n in [(s * t.element_size(), n) for s, n in zip(t.stride(), t.shape) if n > 1 and s] + [(1, t.element_size())]:
            most[c] = most.get(c, 0) + n - 1
    return _solvable(sorted(most.items(), reverse=True), _bytes(b)[1] - 1 - a.data_ptr(), [_STEPS])


def _folded(t: torch.Tensor) -> bool:
    """Whether two elements of ``t`` share their place."""
    dims = sorted((s, n - 1) for s, n in zip(t.stride(), t.shape) if n > 1)
    if not dims or t.numel() == 0:
        return False
    span = 0
    for s, most in dims:
        if s <= span:
            break
        span += s * most
    else:
        return False  # each stride exceeds what the dimensions inside it span
    for k, (s, most) in enumerate(dims):
        # differences of two indexes, here at least 1: s * d summed up is 0
        if s == 0:
            return True
        terms = sorted([(c, 2 * m) for i, (c, m) in enumerate(dims) if i != k and c] + [(s, most - 1)], reverse=True)
        if _solvable(terms, sum(c * m for i, (c, m) in enumerate(dims) if i != k) - s, [_STEPS]):
            return True
    return False


def _check_apart(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor], copied: set[int]) -> None:
    """Raises where a result has a place twice, or shares one with another result or with a gradient that is not the same view.  For pairs with one of the
    ``copied``, of which the native call sees only a copy: it looks at the others itself."""
    places = []
    for i, (g, out) in enumerate(zip(grads, outs)):
        if out.numel() == 0:
            continue
        if i in copied and _folded(out):
            raise ValueError("a result has elements that share their place")
        places.append((*_bytes(out), True, i, out, _column(out)))
        if not (out is g or (out.data_ptr() == g.data_ptr() and out.stride() == g.stride())):
            places.append((*_bytes(g), False, i, g, _column(g)))
    places.sort(key=lambda p: p[:2])
    open_: list[tuple] = []  # those that reach past the place looked at
    for p in places:
        open_ = [q for q in open_ if q[1] > p[0]]
        pitch, begin, end = p[5]
        for q in open_:
            if pitch and q[5][0] == pitch and (q[5][2] <= begin or end <= q[5][1]):
                continue  # columns of one matrix, next to each other: the many pairs of a list that there may be
            if (p[2] or q[2]) and (p[3] in copied or q[3] in copied) and _meet(p[4], q[4]):
                raise ValueError("a result overlaps another tensor")
        open_.append(p)


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


_DTYPE = torch.Tensor.dtype.__get__


def _plain_words(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor] | None, index: int) -> list[int] | None:
    """The kernels' table of a list whose tensors all lie as they take them (most lists: a tensor costs half a microsecond, in place
    a third); ``None`` for others, whatever it is about them."""
    of, codes = torch.Tensor, _lib._DTYPE_CODES
    try:
        if not all(map(of.is_contiguous, grads)) or set(map(of.get_device, grads)) != {index}:
            return None
        words = [0] * (4 * len(grads))  # lbi_gradient of include/lbi_hip.h: four words of 64 bits
        words[0::4] = map(of.data_ptr, grads)
        words[2::4] = map(of.numel, grads)
        types = list(map(_DTYPE, grads))
        words[3::4] = map(codes.__getitem__, types)
        if forward_ad._current_level >= 0 or torch.is_grad_enabled() and torch._C._any_requires_grad(grads, () if outs is None or outs is grads else outs):
            return None
        if outs is None:
            return words
        if outs is grads:
            words[1::4] = words[0::4]
            return words
        if not all(map(of.is_contiguous, outs)) or set(map(of.get_device, outs)) != {index}:
            return None
        if list(map(_DTYPE, outs)) != types or not all(map(of.is_same_size, outs, grads)):
            return None
        words[1::4] = map(of.data_ptr, outs)
        return words
    except (AttributeError, KeyError, RuntimeError, TypeError):
        return None


def _clip(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor] | None, max_norm: float) -> torch.Tensor:
    """``outs``: where the results go (``grads`` itself: in place; ``None``: nowhere, the norm alone)."""
    if not isinstance(grads[0], torch.Tensor) or not grads[0].is_cuda:
        _refuse(grads[:1], "grads", 0)
    index = grads[0].get_device()
    words, held, late, copied = _plain_words(grads, outs, index), [], [], set()
    for i, g in enumerate(grads if words is None else ()):
        to = out = None if outs is None else outs[i]
        _refuse([g], "grads", index)
        if out is not None:
            _refuse([out], "out", index)
            if g.shape != out.shape or out.dtype != g.dtype:
                raise ValueError("out must have the shapes and types of the gradients")
            if out.requires_grad and torch.is_grad_enabled():
                raise RuntimeError("clip_gradients writes tensors that require grad: call it under torch.no_grad()")
        _lib.refuse_graph("gradient_norm" if outs is None else "clip_gradients", g, out)
        if not _flat(g) or not (out is None or out is g or out.stride() == g.stride()):
            g = g.contiguous()
            copied.add(i)
            if out is not None and (out is grads[i] or not out.is_contiguous()):
                to = torch.empty_like(g)
                late.append((out, to))
            # a contiguous `out` of its own is written by the kernel
        held.append((g.data_ptr(), 0 if to is None else to.data_ptr(), g.numel(), _lib.dtype_code(g.dtype), g, to))  # copies live until all is queued
    if words is None:
        words = [word for row in held for word in row[:4]]
    if copied and outs is not None:
        _check_apart(grads, outs, copied)
    count, device = len(grads), grads[0].device
    table = array.array("q", words)
    norm = grads[0].new_empty((), dtype=torch.float32)  # half the time of torch.empty
    lib = _lib.load()
    with _lib.device_guard(device):
        need = lib.lbi_clip_gradients_workspace_bytes(count)
        workspace = grads[0].new_empty(need, dtype=torch.uint8)
        status = lib.lbi_clip_gradients(table.buffer_info()[0], count, max_norm, norm.data_ptr(), workspace.data_ptr(), need, _lib.current_stream_ptr(device))
    _lib.check(status, "lbi_clip_gradients")
    for out, to in late:
        out.copy_(to)
    if outs is not None:
        torch.autograd.graph.increment_version(outs)  # autograd refuses a backward pass that saved what was there before
    return norm


def gradient_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all elements of all ``grads`` (fp32, fp16, bf16, mixed), a scalar tensor of fp32 on their device.
    Squares are added in 64 bits.  An empty list has the norm 0 (on the CPU).  No autograd graph is recorded: tensors that require grad, with
    grad mode on, are refused."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    return _clip(grads, None, math.inf)


def clip_gradients(grads: Sequence[torch.Tensor], max_norm: float, *, out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """``out[i] = grads[i] * min(1, max_norm / (norm + 1e-6))``, ``norm`` the 2-norm over all of ``grads``; in place
    without ``out``.  Returns ``norm``, a scalar tensor of fp32 on the device: nothing here waits for it.

    ``out[i]`` has the shape and type of ``grads[i]`` and is ``grads[i]`` itself or overlaps no gradient and no other
    result, and no two of its elements are one; the same gradient twice in the list counts twice and needs an ``out`` for each.  As
    ``torch.nn.utils.clip_grad_norm_`` does: a norm that is not a number makes every result one, an infinite norm makes
    finite elements 0.  In place and with a norm below the limit, nothing is written.  No
    autograd graph is recorded: tensors that require grad, with grad mode on, are refused."""
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
