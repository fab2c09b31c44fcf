"""The MLP half of a Transformer block, forwards and backwards, on the GPU: the addition to the residual stream with its RMS
norm, and the gated MLP.

    residual_out = hidden + residual;   normed = rmsnorm(residual_out);   out = fc2(up * silu(gate)),  [up | gate] = fc1(normed)

What the reference's block computes in torch (backbones/transformer/block.py:12-23, :66-87, backbones/transformer/mlp.py:10-32, with
the caches of backends/transformer.py:172-188).  The forward functions return what the region pullback reads from a block's cache
(``norm_input``, ``norm_output``, ``fc1_output``, ``down_input``); the pullbacks here are those of a single dense cotangent, parameter
gradients included, where :mod:`.region` pulls a basis of cotangents back through a whole region.

Like the rest of the package these are plain functions with explicit pullbacks and no autograd nodes: forward function or pullback, one that
is given a tensor (a parameter too) that requires grad, with grad mode on, or one with a tangent of forward-mode differentiation, raises
instead of returning a result that is cut off from the graph.
"""
from __future__ import annotations

import torch

from ... import _lib
from .region import _require_cuda, _stream

_PRODUCT_TYPES = (torch.float16, torch.bfloat16)


def _one_device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    device = first.device
    if device.type != "cuda":
        _require_cuda(first)
    for t in others:
        if t is not None and t.device != device:
            _require_cuda(t)
            raise ValueError(f"{what}: tensors must be on one device")


def _norm_types(what: str, branch: torch.dtype, stream: torch.dtype, weight: torch.Tensor) -> torch.Tensor:
    """The weight in a type that the kernels take (the branch's, or fp32 for any other), after a check of the other types."""
    _lib.dtype_code(branch)
    if stream not in (branch, torch.float32):
        raise ValueError(f"{what}: the residual stream must be in the dtype of the branch or fp32")
    return weight if weight.dtype in (branch, torch.float32) else weight.float()


def residual_rmsnorm(hidden: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                     residual_dtype: torch.dtype | None = None, scaled: bool = False) -> tuple[torch.Tensor, ...]:
    """``s = hidden + residual`` and ``y = s * rsqrt(mean(s^2) + eps) * weight`` over the last dimension, in one pass.

    ``hidden, residual [..., D]`` (``residual=None``: zero), ``weight [D]``.  Returns ``(y, s)``: ``y`` in the dtype of ``hidden``,
    ``s`` in ``residual_dtype`` (that of ``residual`` by default, of ``hidden`` without one; of ``hidden`` or fp32).  ``scaled``:
    ``(y8, scales, s)`` instead, ``y8`` in ``torch.float8_e4m3fn`` and ``scales [...]`` in fp32, one a row, ``y = y8 * scales``:
    the row's largest magnitude over 448 (1 for a row of zeros).  Sums are fp32 and each result is rounded once: the norm is that of
    the sum before its rounding to ``residual_dtype``, and a ``residual`` of another type than that enters the sum as it is (in fp32, with
    one more pass that rounds ``s``)."""
    if hidden.dim() < 1 or weight.shape != hidden.shape[-1:]:
        raise ValueError("residual_rmsnorm: hidden must be [..., D] and weight [D]")
    if residual is not None and residual.shape != hidden.shape:
        raise ValueError("residual_rmsnorm: residual must be shaped like hidden")
    _one_device("residual_rmsnorm", hidden, residual, weight)
    _lib.refuse_graph("residual_rmsnorm", hidden, residual, weight)
    branch = hidden.dtype
    stream = residual_dtype or (branch if residual is None else residual.dtype)
    weight = _norm_types("residual_rmsnorm", branch, stream, weight).contiguous()
    hidden = hidden.contiguous()
    held = stream if residual is None or residual.dtype == stream else torch.float32  # what the kernel reads and writes
    if residual is not None:
        residual = (residual if residual.dtype == held else residual.to(held)).contiguous()
    total = torch.empty_like(hidden, dtype=held)
    normed = torch.empty_like(hidden, dtype=torch.float8_e4m3fn) if scaled else torch.empty_like(hidden)
    scales = hidden.new_empty(hidden.shape[:-1], dtype=torch.float32) if scaled else None
    count, width = hidden.numel(), hidden.shape[-1]
    if count:
        with _lib.device_guard(hidden.device):
            status = _lib.load().lbi_residual_rmsnorm(
                hidden.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(), normed.data_ptr(),
                total.data_ptr(), None if scales is None else scales.data_ptr(), count // width, width, eps,
                _lib.dtype_code(branch), _lib.dtype_code(held), _lib.dtype_code(weight.dtype), _stream(hidden))
        _lib.check(status, "lbi_residual_rmsnorm")
    elif scales is not None:
        scales.fill_(1.0)
    if held is not stream:
        total = total.to(stream)
    return (normed, scales, total) if scales is not None else (normed, total)


def residual_rmsnorm_pullback(g_normed: torch.Tensor, residual_out: torch.Tensor, weight: torch.Tensor, eps: float, *,
                              g_residual: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The cotangents of :func:`residual_rmsnorm` from ``g_normed`` (of its ``y``) and ``g_residual`` (of its ``s``; ``None``: zero),
    both shaped like ``residual_out``, the ``s`` that it returned.

    Returns ``(g_hidden, g_residual_in, g_weight)``: the cotangent of both inputs in the dtype of ``g_normed`` and in that of
    ``residual_out`` (one and the same tensor where these are the same), and the weight's gradient, fp32 ``[D]``, summed over all rows
    in a fixed order.  ``g_residual`` is in the dtype of ``residual_out``."""
    if g_normed.dim() < 1 or residual_out.shape != g_normed.shape or weight.shape != g_normed.shape[-1:]:
        raise ValueError("residual_rmsnorm_pullback: g_normed and residual_out must be [..., D] and weight [D]")
    if g_residual is not None and (g_residual.shape != g_normed.shape or g_residual.dtype != residual_out.dtype):
        raise ValueError("residual_rmsnorm_pullback: g_residual must have the shape and dtype of residual_out")
    _one_device("residual_rmsnorm_pullback", g_normed, residual_out, weight, g_residual)
    _lib.refuse_graph("residual_rmsnorm_pullback", g_normed, residual_out, weight, g_residual)
    branch, stream = g_normed.dtype, residual_out.dtype
    weight = _norm_types("residual_rmsnorm_pullback", branch, stream, weight).contiguous()
    g_normed, residual_out = g_normed.contiguous(), residual_out.contiguous()
    if g_residual is not None:
        g_residual = g_residual.contiguous()
    g_stream = torch.empty_like(residual_out)
    g_hidden = g_stream if stream == branch else torch.empty_like(g_normed)
    width = int(g_normed.shape[-1])
    g_weight = g_normed.new_empty(width, dtype=torch.float32)
    if not width:
        return g_hidden, g_stream, g_weight
    rows = g_normed.numel() // width
    lib = _lib.load()
    with _lib.device_guard(g_normed.device):
        need = int(lib.lbi_residual_rmsnorm_pullback_workspace_bytes(rows, width))
        workspace = g_normed.new_empty(max(need, 16), dtype=torch.uint8)
        status = lib.lbi_residual_rmsnorm_pullback(
            g_normed.data_ptr(), residual_out.data_ptr(), None if g_residual is None else g_residual.data_ptr(), weight.data_ptr(),
            None if g_hidden is g_stream else g_hidden.data_ptr(), g_stream.data_ptr(), g_weight.data_ptr(), workspace.data_ptr(), need,
            rows, width, float(eps), _lib.dtype_code(branch), _lib.dtype_code(stream), _lib.dtype_code(weight.dtype), _stream(g_normed))
    _lib.check(status, "lbi_residual_rmsnorm_pullback")
    return g_hidden, g_stream, g_weight


def _check_mlp(what: str, x: torch.Tensor, fc1_weight: torch.Tensor, fc2_weight: torch.Tensor) -> tuple[int, int, int, int]:
    """``(rows, D, hidden, width)``."""
    if x.dtype not in _PRODUCT_TYPES:
        raise TypeError(f"{what}: unsupported dtype {x.dtype}; expected float16 or bfloat16")
    if fc1_weight.dim() != 2 or fc2_weight.dim() != 2 or fc1_weight.shape[0] != 2 * fc2_weight.shape[1]:
        raise ValueError(f"{what}: fc1_weight must be [2 * hidden, D] and fc2_weight [width, hidden]")
    if x.dim() < 1 or x.shape[-1] != fc1_weight.shape[1]:
        raise ValueError(f"{what}: x must be [..., D] for fc1_weight [2 * hidden, D]")
    width, hidden = fc2_weight.shape
    dim = int(x.shape[-1])
    if not dim or not hidden or not width:
        raise ValueError(f"{what}: widths must not be 0")
    return x.numel() // dim, dim, int(hidden), int(width)


def _ready(t: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor | None:
    """``t`` in ``dtype``, contiguous and on the kernels' 16-byte grid."""
    if t is None or (t.dtype == dtype and t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    t = t.detach().to(dtype).contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def gated_mlp(x: torch.Tensor, fc1_weight: torch.Tensor, fc2_weight: torch.Tensor, fc1_bias: torch.Tensor | None = None,
              fc2_bias: torch.Tensor | None = None, *, keep: bool = False):
    """``out = fc2(up * silu(gate))``, ``[up | gate] = fc1(x)``, for ``x [..., D]`` in fp16 or bf16, ``fc1_weight [2 * hidden, D]``,
    ``fc2_weight [width, hidden]`` and biases ``[2 * hidden]`` and ``[width]``; parameters of another type are cast to that of ``x``.

    Returns ``out [..., width]`` in the dtype of ``x``; with ``keep`` ``(out, fc1_output [..., 2 * hidden], down_input [..., hidden])``,
    what :func:`gated_mlp_vjp` and the region pullback read.  Sums, biases and the activation are fp32; ``down_input``, the
    operand of the second product, is the one rounding in between.  Widths that are no multiples of 8 run on padded copies, a pass over
    the operands and one over the results."""
    rows, dim, hidden, width = _check_mlp("gated_mlp", x, fc1_weight, fc2_weight)
    if (fc1_bias is not None and fc1_bias.shape != (2 * hidden,)) or (fc2_bias is not None and fc2_bias.shape != (width,)):
        raise ValueError("gated_mlp: fc1_bias must be [2 * hidden] and fc2_bias [width]")
    _one_device("gated_mlp", x, fc1_weight, fc2_weight, fc1_bias, fc2_bias)
    _lib.refuse_graph("gated_mlp", x, fc1_weight, fc2_weight, fc1_bias, fc2_bias)
    dtype, outer = x.dtype, x.shape[:-1]
    out, down = x.new_empty(*outer, width), x.new_empty(*outer, hidden)
    fc1_output = x.new_empty(*outer, 2 * hidden) if keep else None
    if rows:
        x, fc1_weight, fc2_weight = _ready(x, dtype), _ready(fc1_weight, dtype), _ready(fc2_weight, dtype)
        fc1_bias, fc2_bias = _ready(fc1_bias, dtype), _ready(fc2_bias, dtype)
        lib = _lib.load()
        with _lib.device_guard(x.device):
            need = lib.lbi_gated_mlp_workspace_bytes(rows, dim, hidden, width)
            workspace = x.new_empty(need, dtype=torch.uint8) if need else None
            status = lib.lbi_gated_mlp(
                x.data_ptr(), fc1_weight.data_ptr(), None if fc1_bias is None else fc1_bias.data_ptr(), fc2_weight.data_ptr(),
                None if fc2_bias is None else fc2_bias.data_ptr(), None if fc1_output is None else fc1_output.data_ptr(),
                down.data_ptr(), out.data_ptr(), None if workspace is None else workspace.data_ptr(), need, rows, dim, hidden, width,
                _lib.dtype_code(dtype), _stream(x))
        _lib.check(status, "lbi_gated_mlp")
    return (out, fc1_output, down) if keep else out


def gated_mlp_vjp(g_out: torch.Tensor, x: torch.Tensor, fc1_output: torch.Tensor, down_input: torch.Tensor, fc1_weight: torch.Tensor,
                  fc2_weight: torch.Tensor, *, bias: bool = False) -> tuple[torch.Tensor, ...]:
    """The cotangents of :func:`gated_mlp` at ``x`` for ``g_out [..., width]``, from the ``fc1_output`` and ``down_input`` that it
    returned with ``keep``.

    Returns ``(g_x, g_fc1_weight, g_fc2_weight)``, with ``bias`` also ``g_fc1_bias`` and ``g_fc2_bias``, all in the dtype of ``x`` (which is
    that of ``g_out`` and the caches).  Sums are fp32; the cotangent of ``fc1_output`` is the one rounding in between."""
    rows, dim, hidden, width = _check_mlp("gated_mlp_vjp", x, fc1_weight, fc2_weight)
    outer, dtype = x.shape[:-1], x.dtype
    for name, t, extent in (("g_out", g_out, width), ("fc1_output", fc1_output, 2 * hidden), ("down_input", down_input, hidden)):
        if t.shape != (*outer, extent) or t.dtype != dtype:
            raise ValueError(f"gated_mlp_vjp: {name} must be {(*outer, extent)} in the dtype of x")
    _one_device("gated_mlp_vjp", x, g_out, fc1_output, down_input, fc1_weight, fc2_weight)
    _lib.refuse_graph("gated_mlp_vjp", x, g_out, fc1_output, down_input, fc1_weight, fc2_weight)
    if not rows:
        empty = [torch.zeros_like(x), x.new_zeros(fc1_weight.shape), x.new_zeros(fc2_weight.shape)]
        return tuple(empty + [x.new_zeros(2 * hidden), x.new_zeros(width)] if bias else empty)
    g_out, x, fc1_output, down_input = _ready(g_out, dtype), _ready(x, dtype), _ready(fc1_output, dtype), _ready(down_input, dtype)
    fc1_weight, fc2_weight = _ready(fc1_weight, dtype), _ready(fc2_weight, dtype)
    g_x, g_fc1, g_fc2 = torch.empty_like(x), x.new_empty(2 * hidden, dim), x.new_empty(width, hidden)
    g_fc1_bias, g_fc2_bias = (x.new_empty(2 * hidden), x.new_empty(width)) if bias else (None, None)
    lib = _lib.load()
    with _lib.device_guard(x.device):
        need = lib.lbi_gated_mlp_vjp_workspace_bytes(rows, dim, hidden, width)
        workspace = x.new_empty(need, dtype=torch.uint8)
        status = lib.lbi_gated_mlp_vjp(
            g_out.data_ptr(), x.data_ptr(), fc1_output.data_ptr(), down_input.data_ptr(), fc1_weight.data_ptr(), fc2_weight.data_ptr(),
            g_x.data_ptr(), g_fc1.data_ptr(), g_fc2.data_ptr(), g_fc1_bias.data_ptr() if bias else None,
            g_fc2_bias.data_ptr() if bias else None, workspace.data_ptr(), need, rows, dim, hidden, width, _lib.dtype_code(dtype), _stream(x))
    _lib.check(status, "lbi_gated_mlp_vjp")
    return (g_x, g_fc1, g_fc2, g_fc1_bias, g_fc2_bias) if bias else (g_x, g_fc1, g_fc2)


__all__ = ["gated_mlp", "gated_mlp_vjp", "residual_rmsnorm", "residual_rmsnorm_pullback"]
