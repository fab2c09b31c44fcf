"""Plain restatements of a linear-attention block's mixer half, for tests: rotary positions, linear attention by its recurrence, and the norms
behind and before a block with gate and residual scale.  Differentiable, in the type of their arguments (64 bits in the tests)."""
from __future__ import annotations

import torch


def rotary_turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """``x [..., T, Dh]``, tables ``[..., T, R / 2]`` (broadcast)."""
    half = cos.shape[-1]
    out = x.clone()
    for i in range(half):
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        out[..., first] = x[..., first] * cos[..., i] - x[..., second] * sin[..., i]
        out[..., second] = x[..., first] * sin[..., i] + x[..., second] * cos[..., i]
    return out


def rotary_heads(qkv, cos, sin, *, n_heads, n_kv_heads, interleaved=False, positions=None):
    bsz, seqlen, width = qkv.shape
    head_dim = width // (n_heads + 2 * n_kv_heads)
    x = qkv.view(bsz, seqlen, -1, head_dim).transpose(1, 2)
    at = torch.arange(seqlen).expand(bsz, seqlen) if positions is None else positions.expand(bsz, seqlen)
    turned = rotary_turn(x[:, :n_heads + n_kv_heads], cos[at][:, None], sin[at][:, None], interleaved)
    return turned[:, :n_heads], turned[:, n_heads:], x[:, n_heads + n_kv_heads:]


def linear_attention(q, k, v, log_decay, *, scale, state=None, lengths=None):
    """One token after the other.  ``(out [B, H, T, Dv], state [B, H, Dk, Dv])``."""
    bsz, heads, seqlen, _ = q.shape
    group = heads // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    decay = log_decay.to(q.dtype).exp()[:, None, None]
    s = torch.zeros(bsz, heads, q.shape[-1], v.shape[-1], dtype=q.dtype) if state is None else state
    rows = []
    for t in range(seqlen):
        on = torch.ones(bsz, dtype=torch.bool) if lengths is None else t < lengths
        on = on[:, None, None, None]
        # torch.where with clean values on both sides: what lies behind a sequence may be anything
        kt, vt, qt = (torch.where(on[..., 0], x[:, :, t], torch.zeros((), dtype=q.dtype)) for x in (k, v, q))
        s = torch.where(on, decay * s + kt[..., None] * vt[..., None, :], s)
        rows.append(scale * torch.where(on[..., 0], (qt[..., None, :] @ s)[..., 0, :], torch.zeros((), dtype=q.dtype)))
    out = torch.stack(rows, 2) if rows else q.new_zeros(bsz, heads, 0, v.shape[-1])
    return out, s


def rounded_operands(a, b, c, log_decay, first=None, *, lengths=None, reverse=False, shift=0):
    """What rounding of the operands can change in ``out_i = sum over j <= i of l^(i-j) (a_i . b_j) c_j`` (from the last token that counts, with
    ``reverse``), relative to half a step of the operand type: the magnitudes of the decayed scores of each 64 tokens against ``|c|``, and of ``a``
    against the state in front of the 64.  ``[B, H, T, Dc]`` in 64 bits."""
    bsz, heads, seqlen, _ = a.shape
    decay = log_decay.double().exp()
    most = torch.zeros(bsz, heads, seqlen, c.shape[-1], dtype=torch.float64)
    for n in range(bsz):
        count = seqlen if lengths is None else int(lengths[n])
        order = torch.arange(count)
        if reverse:
            order = order.flip(0)
        for h in range(heads):
            x = torch.zeros(a.shape[-1], c.shape[-1], dtype=torch.float64) if first is None else first[n, h].double()
            for from_ in range(0, count, 64):
                at = order[from_:from_ + 64]
                aa, bb, cc = a[n, h, at].double(), b[n, h, at].double(), c[n, h, at].double()
                i = torch.arange(len(at), dtype=torch.float64)
                apart = i[:, None] - i
                pairs = (aa @ bb.T) * torch.where(apart >= 0, decay[h] ** apart.clamp(min=0), 0.0)
                most[n, h, at] = pairs.abs() @ cc.abs() + decay[h] ** (i + 1 - shift)[:, None] * (aa.abs() @ x.abs())
                x = decay[h] ** len(at) * x + (bb * decay[h] ** (len(at) - 1 - i + shift)[:, None]).T @ cc
    return most


def gated_residual_rmsnorm(branch, residual, post_weight, weight, eps, *, gate=None, residual_scale=1.0):
    unit = branch / (branch.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    total = residual_scale * residual + unit * post_weight * (1.0 if gate is None else gate)
    return total / (total.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight, total
