"""The mixer half of a Transformer block whose attention is linear, on the GPU: rotary positions and linear attention with a decay for each
head, forwards and backwards.

    q, k, v = rotary_heads(in_proj(x));   S_t = exp(log_decay) S_{t-1} + k_t v_t^T,   out_t = scale q_t S_t

Stands beside the softmax attention of this package (``attention_input_pullback_basis``, ``attn_qkv_pullback``): the same tensors, heads and
bases of cotangents, for a mixer whose state does not grow with the context.  A head's decay is a constant of the layer, without a gradient; mixers whose decay depends
on the token, as those of the reference's second and third backbone (whose input pullback for a basis is a stub there, cuda/mamba3/__init__.py:4-8), are
not served by it.  The turn is that of the reference's apply_rope
(backbones/transformer/rope.py:6-34), with part of a head, positions and stretched angles beside it.

Plain functions with explicit pullbacks and no autograd nodes, as in :mod:`.block`: one that is given a tensor that requires grad, with
grad mode on, or one with a tangent of forward-mode differentiation, raises.  No function synchronises; each can be captured into a graph.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ... import _lib
from .region import _require_cuda, _stream

_ATTENTION_TYPES = (torch.float16, torch.bfloat16)
_WHOLE_TYPES = (torch.int32, torch.int64)


def _one_device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    for t in (first, *others):
        if t is not None and t.device != first.device:
            _require_cuda(t)
            raise ValueError(f"{what}: tensors must be on one device")
    _require_cuda(first)


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def rotary_tables(length: int, rotary_dim: int, base: float = 10000.0, *, device: torch.device | str, factor: float = 1.0,
                  original_length: int | None = None, ramp: tuple[float, float] = (1.0, 32.0),
                  magnitude: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """``cos`` and ``sin`` ``[length, rotary_dim / 2]`` in fp32 of the angles ``position * base ** (-2 i / rotary_dim)``, computed in 64 bits:
    far positions lose no digits.  Built once and kept by the caller.

    For contexts ``factor`` times as long as those trained on: every angle is divided by ``factor``; with ``original_length`` (the length trained on) only the
    slow ones are, by how many turns they make over that length: those of fewer than ``ramp[0]`` are divided, those of more than ``ramp[1]`` are left,
    and in between the two are blended linearly.  ``magnitude`` multiplies both tables (and so scores by its square)."""
    if length < 0 or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_tables: length must not be negative and rotary_dim even")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor) and math.isfinite(magnitude)):
        raise ValueError("rotary_tables: base and factor must be positive, and magnitude finite")
    if original_length is not None and not (original_length > 0 and ramp[0] < ramp[1]):
        raise ValueError("rotary_tables: original_length must be positive and ramp rising")
    half = rotary_dim // 2
    frequency = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) * 2 / max(rotary_dim, 1))
    if original_length is None:
        frequency = frequency / factor
    else:
        turns = original_length * frequency / (2 * math.pi)
        kept = ((turns - ramp[0]) / (ramp[1] - ramp[0])).clamp(0, 1)
        frequency = frequency * (kept + (1 - kept) / factor)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * frequency
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()


def _check_tables(what: str, cos: torch.Tensor, sin: torch.Tensor, head_dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    if cos.dim() != 2 or sin.shape != cos.shape or 2 * cos.shape[1] > head_dim:
        raise ValueError(f"{what}: cos and sin must be [positions, rotary_dim / 2] with rotary_dim at most the head dimension {head_dim}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"{what}: cos and sin must be fp32")
    return cos.contiguous(), sin.contiguous()


def _check_positions(what: str, positions: torch.Tensor | None, bsz: int, seqlen: int, table: int) -> torch.Tensor | None:
    if positions is None:
        if table < seqlen:
            raise ValueError(f"{what}: tables of {table} positions for {seqlen} tokens")
        return None
    if positions.dtype not in _WHOLE_TYPES:
        raise ValueError(f"{what}: positions must be int32 or int64")
    if positions.shape not in ((seqlen,), (bsz, seqlen)):
        raise ValueError(f"{what}: positions must be [T] or [B, T]")
    return (positions if positions.dim() == 2 else positions.expand(bsz, seqlen)).contiguous()


def rotary_heads(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, n_heads: int, n_kv_heads: int, interleaved: bool = False,
                 positions: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The heads of the packed projection ``qkv [B, T, (H + 2 Hkv) Dh]``: ``q [B, H, T, Dh]`` and ``k [B, Hkv, T, Dh]``, contiguous, the first
    ``R`` elements of each head turned by its position's angles, and ``v [B, Hkv, T, Dh]``, a view of ``qkv``.

    ``cos, sin [positions, R / 2]`` (:func:`rotary_tables`), ``R <= Dh``; pairs are ``(i, i + R / 2)``, or ``(2 i, 2 i + 1)`` if ``interleaved``.
    ``positions`` (int32 or int64, ``[T]`` or ``[B, T]``; default ``0 ... T-1``) are rows of the tables; one outside turns its token's ``R``
    elements into NaN.  fp32, fp16 or bf16; computed in fp32 and rounded once."""
    what = "rotary_heads"
    if n_heads < 1 or n_kv_heads < 1 or n_heads % n_kv_heads:
        raise ValueError("n_heads must be divisible by n_kv_heads")
    if qkv.dim() != 3 or qkv.shape[2] == 0 or qkv.shape[2] % (n_heads + 2 * n_kv_heads):
        raise ValueError(f"{what}: qkv must be [B, T, (n_heads + 2 * n_kv_heads) * head_dim]")
    bsz, seqlen, width = qkv.shape
    head_dim = width // (n_heads + 2 * n_kv_heads)
    dtype = _lib.dtype_code(qkv.dtype)
    cos, sin = _check_tables(what, cos, sin, head_dim)
    positions = _check_positions(what, positions, bsz, seqlen, cos.shape[0])
    _one_device(what, qkv, cos, sin, positions)
    _lib.refuse_graph(what, qkv, cos, sin)
    qkv = _dense_rows(qkv)
    q, k = qkv.new_empty(bsz, n_heads, seqlen, head_dim), qkv.new_empty(bsz, n_kv_heads, seqlen, head_dim)
    step_b, step_t, _ = qkv.stride()
    v = qkv.as_strided((bsz, n_kv_heads, seqlen, head_dim), (step_b, head_dim, step_t, 1), qkv.storage_offset() + (n_heads + n_kv_heads) * head_dim)
    if q.numel():
        with _lib.device_guard(qkv.device):
            status = _lib.load().lbi_rotary(
                qkv.data_ptr(), cos.data_ptr(), sin.data_ptr(), None if positions is None else positions.data_ptr(), q.data_ptr(), k.data_ptr(),
                bsz, seqlen, n_heads, n_kv_heads, head_dim, 2 * cos.shape[1], cos.shape[0], step_b, step_t,
                int(positions is not None and positions.dtype == torch.int64), int(bool(interleaved)), dtype, _stream(qkv))
        _lib.check(status, "lbi_rotary")
    return q, k, v


def rotary_heads_pullback(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, n_kv_heads: int,
                          interleaved: bool = False, positions: torch.Tensor | None = None) -> torch.Tensor:
    """The cotangent ``[B, P, T, (H + 2 Hkv) Dh]`` of :func:`rotary_heads`'s ``qkv`` for ``P`` directions, from ``dq [B, P, H, T, Dh]`` and
    ``dk, dv`` of ``H`` heads (as the attention pullbacks give them: those of heads that share a key or value are added up, in fp32, before the one
    rounding) or of ``Hkv``."""
    what = "rotary_heads_pullback"
    if dq.dim() != 5 or dk.dim() != 5 or dv.shape != dk.shape:
        raise ValueError(f"{what}: dq, dk, dv must be [B, P, heads, T, Dh]")
    bsz, basis, heads, seqlen, head_dim = dq.shape
    if heads < 1 or n_kv_heads < 1 or heads % n_kv_heads:
        raise ValueError("n_heads must be divisible by n_kv_heads")
    kv_heads = dk.shape[2]
    if dk.shape != (bsz, basis, kv_heads, seqlen, head_dim) or kv_heads not in (heads, n_kv_heads) or head_dim < 1:
        raise ValueError(f"{what}: dk and dv must be shaped like dq, with {heads} or {n_kv_heads} heads")
    if dk.dtype != dq.dtype or dv.dtype != dq.dtype:
        raise ValueError(f"{what}: dq, dk, dv must have one dtype")
    dtype = _lib.dtype_code(dq.dtype)
    cos, sin = _check_tables(what, cos, sin, head_dim)
    positions = _check_positions(what, positions, bsz, seqlen, cos.shape[0])
    _one_device(what, dq, dk, dv, cos, sin, positions)
    _lib.refuse_graph(what, dq, dk, dv, cos, sin)
    dq, dk, dv = dq.contiguous(), dk.contiguous(), dv.contiguous()
    out = dq.new_empty(bsz, basis, seqlen, (heads + 2 * n_kv_heads) * head_dim)
    if out.numel():
        with _lib.device_guard(dq.device):
            status = _lib.load().lbi_rotary_pullback(
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), cos.data_ptr(), sin.data_ptr(), None if positions is None else positions.data_ptr(),
                out.data_ptr(), bsz, basis, seqlen, heads, n_kv_heads, kv_heads, head_dim, 2 * cos.shape[1], cos.shape[0],
                int(positions is not None and positions.dtype == torch.int64), int(bool(interleaved)), dtype, _stream(dq))
        _lib.check(status, "lbi_rotary_pullback")
    return out


def _check_attention(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float, tokens: int) -> None:
    """Shapes ``[B, H, (T,) D]`` (``tokens``: with ``T``), types and what no kernel takes."""
    of_q, of_k, of_v = q.shape, k.shape, v.shape
    if len(of_q) != 3 + tokens or len(of_k) != len(of_q) or of_v[:-1] != of_k[:-1] or of_k[0] != of_q[0] or of_k[2:] != of_q[2:]:
        raise ValueError(f"{what}: q must be [B, H, {'T, ' * tokens}Dk], k [B, Hkv, {'T, ' * tokens}Dk] and v [B, Hkv, {'T, ' * tokens}Dv]")
    heads, kv_heads = of_q[1], of_k[1]
    if not heads or not kv_heads or heads % kv_heads:
        raise ValueError(f"{what}: the heads of q must be a multiple of those of k and v")
    if not of_q[-1] or not of_v[-1]:
        raise ValueError(f"{what}: head dimensions must not be 0")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"{what}: q, k and v must have one dtype")
    if log_decay.shape != (heads,) or log_decay.dtype != torch.float32:
        raise ValueError(f"{what}: log_decay must be [H] in fp32")
    if not 2.0 ** -128 < abs(ctypes.c_float(scale).value) < math.inf:  # NaN is neither
        raise ValueError(f"{what}: scale must be finite and not zero, and so must its inverse, in fp32")


def _check_states(what: str, name: str, t: torch.Tensor | None, shape: tuple[int, ...]) -> torch.Tensor | None:
    if t is None:
        return None
    if t.shape != shape or t.dtype != torch.float32:
        raise ValueError(f"{what}: {name} must be {list(shape)} in fp32")
    return t.contiguous()


def _check_lengths(what: str, lengths: torch.Tensor | None, bsz: int) -> torch.Tensor | None:
    if lengths is None:
        return None
    if lengths.shape != (bsz,) or lengths.dtype not in _WHOLE_TYPES:
        raise ValueError(f"{what}: lengths must be [B] in int32 or int64")
    return lengths.contiguous()


def _pointer(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


_NO_STRIDES = (0, 0, 0, 0)


def _call(q, k, v, log_decay, scale, state, lengths, *, basis=1, out=None, state_out=None, g_out=None, g_state=None, grads=(None, None, None),
          d_state=None) -> bytes:
    """``lbi_linear_attention_call`` of include/lbi_hip.h, as bytes."""
    bsz, heads, seqlen, dk = q.shape
    _, kv_heads, _, dv = v.shape
    return _lib.pack_linear_attention_call(
        bsz, basis, heads, kv_heads, seqlen, dk, dv, q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
        log_decay.data_ptr(), _pointer(state), _pointer(lengths), _pointer(out), *(_NO_STRIDES[:3] if out is None else out.stride()[:3]),
        _pointer(state_out), _pointer(g_out), *(_NO_STRIDES if g_out is None else g_out.stride()[:4]), _pointer(g_state), _pointer(grads[0]),
        _pointer(grads[1]), _pointer(grads[2]), _pointer(d_state), scale, _lib.dtype_code(q.dtype), lengths is not None and lengths.dtype == torch.int64)


def _attention_types(what: str, q: torch.Tensor) -> None:
    if q.dtype not in _ATTENTION_TYPES:
        raise TypeError(f"{what}: unsupported dtype {q.dtype}; expected float16 or bfloat16")


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *, scale: float,
                     state: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                     return_state: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``out_t = scale q_t S_t`` with ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T`` and ``S_{-1} = state`` (zero by default).

    ``q [B, H, T, Dk]``, ``k [B, Hkv, T, Dk]``, ``v [B, Hkv, T, Dv]`` in fp16 or bf16, of any strides whose last one is 1; ``Hkv`` divides ``H`` and neighbouring
    heads share; ``Dk, Dv <= 128``.  ``log_decay [H]`` in fp32 is the layer's constant, 0 or less.  ``scale`` and its inverse are finite in fp32.  ``lengths [B]`` (int32 or int64; clamped to
    ``0 ... T``): the tokens of each sequence that count; those behind them are not read, and the rows of ``out`` there are zero.

    Returns ``(out, S)``: ``out [B, H, T, Dv]`` in the dtype of ``q``, laid out as ``[B, T, H, Dv]`` (what an output projection reads, without a copy), and
    the state ``[B, H, Dk, Dv]`` in fp32 after each sequence's last token, for :func:`linear_attention_step` or the next piece of the context (``None``
    unless ``return_state``).  Sums are fp32; the decayed scores and a copy of the state are rounded to the dtype as operands, so ``out`` is
    off by about 1.4 times what rounding it once would be (calls of up to 64 tokens round it once).  A value that is
    not finite reaches the rows of its 64 tokens (those from a multiple of 64 on; in the pullback's ``dk`` and ``dv`` counted back from the last token),
    earlier ones among them."""
    what = "linear_attention"
    _check_attention(what, q, k, v, log_decay, scale, 1)
    _attention_types(what, q)
    bsz, heads, seqlen, dk = q.shape
    dv = v.shape[-1]
    state = _check_states(what, "state", state, (bsz, heads, dk, dv))
    lengths = _check_lengths(what, lengths, bsz)
    _one_device(what, q, k, v, log_decay, state, lengths)
    _lib.refuse_graph(what, q, k, v, log_decay, state)
    q, k, v, log_decay = _dense_rows(q), _dense_rows(k), _dense_rows(v), log_decay.contiguous()
    out = q.new_empty_strided((bsz, heads, seqlen, dv), (seqlen * heads * dv, dv, heads * dv, 1))
    state_out = q.new_empty(bsz, heads, dk, dv, dtype=torch.float32) if return_state else None
    lib = _lib.load()
    with _lib.device_guard(q.device):
        call = _call(q, k, v, log_decay, scale, state, lengths, out=out, state_out=state_out)
        need = lib.lbi_linear_attention_workspace_bytes(call)
        workspace = q.new_empty(need, dtype=torch.uint8) if need else None
        status = lib.lbi_linear_attention(call, _pointer(workspace), need, _stream(q))
    _lib.check(status, "lbi_linear_attention")
    return out, state_out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *, scale: float,
                          active: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each sequence through :func:`linear_attention`: ``q [B, H, Dk]``, ``k [B, Hkv, Dk]``, ``v [B, Hkv, Dv]`` in fp32, fp16 or bf16, and
    ``state [B, H, Dk, Dv]``, fp32 and contiguous, which is updated in place and shares memory with none of them.  ``active [B]`` (bool): sequences that have no token keep their state
    and get zeros.  Returns ``out [B, H, Dv]``; arithmetic is fp32."""
    what = "linear_attention_step"
    _check_attention(what, q, k, v, log_decay, scale, 0)
    bsz, heads, dk = q.shape
    dv = v.shape[-1]
    if state.shape != (bsz, heads, dk, dv) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{what}: state must be {[bsz, heads, dk, dv]} in fp32, contiguous")
    if active is not None and (active.shape != (bsz,) or active.dtype != torch.bool):
        raise ValueError(f"{what}: active must be [B] in bool")
    dtype = _lib.dtype_code(q.dtype)
    _one_device(what, q, k, v, log_decay, state, active)
    _lib.refuse_graph(what, q, k, v, log_decay, state)
    q, k, v, log_decay = q.contiguous(), k.contiguous(), v.contiguous(), log_decay.contiguous()
    active = None if active is None else active.contiguous()
    out = q.new_empty(bsz, heads, dv)
    if bsz:
        with _lib.device_guard(q.device):
            status = _lib.load().lbi_linear_attention_step(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), state.data_ptr(), _pointer(active), out.data_ptr(), bsz, heads,
                k.shape[1], dk, dv, float(scale), dtype, _stream(q))
        _lib.check(status, "lbi_linear_attention_step")
        torch.autograd.graph.increment_version(state)
    return out


def linear_attention_input_pullback_basis(
        q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, output_cotangent_basis: torch.Tensor, log_decay: torch.Tensor, *, scale: float,
        state: torch.Tensor | None = None, g_state: torch.Tensor | None = None,
        lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """The cotangents of :func:`linear_attention`'s inputs for ``P`` directions (``P = 1``: a training step's), from
    ``output_cotangent_basis [B, P, H, T, Dv]`` of its ``out`` and ``g_state [B, P, H, Dk, Dv]`` (fp32; zero by default) of the state that it returned.

    Returns ``dq, dk [B, P, H, T, Dk]`` and ``dv [B, P, H, T, Dv]``, contiguous, in the dtype of ``q``, and the cotangent ``[B, P, H, Dk, Dv]`` of
    ``state`` (``None`` if no ``state`` was given).  Where heads share ``k`` and ``v`` there is a ``dk`` and ``dv`` for each query head, as
    ``attention_input_pullback_basis`` has them: :func:`rotary_heads_pullback` adds them up.  Nothing is kept from the forward pass; the states
    are recomputed.  Types, strides, ``lengths`` (rows behind them are zero) and roundings as there, and in bf16 without ``state`` the decayed values that a
    state adds up have 16 significant bits instead of 24; ``log_decay`` is a constant."""
    what = "linear_attention_input_pullback_basis"
    _check_attention(what, q, k, v, log_decay, scale, 1)
    _attention_types(what, q)
    bsz, heads, seqlen, dk = q.shape
    dv = v.shape[-1]
    g = output_cotangent_basis
    if g.dim() != 5 or g.shape[0] != bsz or g.shape[2:] != (heads, seqlen, dv) or g.dtype != q.dtype:
        raise ValueError(f"{what}: output_cotangent_basis must be [B, P, H, T, Dv] in the dtype of q")
    basis = g.shape[1]
    state = _check_states(what, "state", state, (bsz, heads, dk, dv))
    g_state = _check_states(what, "g_state", g_state, (bsz, basis, heads, dk, dv))
    lengths = _check_lengths(what, lengths, bsz)
    _one_device(what, q, k, v, g, log_decay, state, g_state, lengths)
    _lib.refuse_graph(what, q, k, v, g, log_decay, state, g_state)
    q, k, v, g, log_decay = _dense_rows(q), _dense_rows(k), _dense_rows(v), _dense_rows(g), log_decay.contiguous()
    grads = tuple(q.new_empty(bsz, basis, heads, seqlen, width) for width in (dk, dk, dv))
    d_state = None if state is None else q.new_empty(bsz, basis, heads, dk, dv, dtype=torch.float32)
    lib = _lib.load()
    with _lib.device_guard(q.device):
        call = _call(q, k, v, log_decay, scale, state, lengths, basis=basis, g_out=g, g_state=g_state, grads=grads, d_state=d_state)
        need = lib.lbi_linear_attention_pullback_workspace_bytes(call)
        workspace = q.new_empty(need, dtype=torch.uint8) if need else None
        status = lib.lbi_linear_attention_pullback(call, _pointer(workspace), need, _stream(q))
    _lib.check(status, "lbi_linear_attention_pullback")
    return (*grads, d_state)


__all__ = ["linear_attention", "linear_attention_input_pullback_basis", "linear_attention_step", "rotary_heads", "rotary_heads_pullback",
           "rotary_tables"]
