"""The MLP half of a Transformer block and gradient clipping in 64 bits, each result with a bound of how far a kernel may be from it.
TEST INFRASTRUCTURE ONLY, as the rest of this package.

Bounds are worst cases by arithmetic, element by element.  ``U`` is half a step of fp32 (2^-24).  A sum of n products in fp32, in any order,
is off by at most n 2U times the sum of the magnitudes (2U an addition: the matrix cores need not round to nearest).  A result stored in
type t is off by half a step of t, ``finfo(t).eps / 2``, and below its normal numbers by half the smallest one.  The sums of
squares of a norm are chains of at most 32 elements a thread and 10 exchanges; the square root halves their error.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def stored(value: torch.Tensor, error: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """``value``, computed with ``error``, rounded to ``dtype``."""
    info = torch.finfo(dtype)
    half = info.eps / 2
    return value, error * (1 + half) + half * value.abs() + info.smallest_normal * info.eps / 2


def assert_near(got: torch.Tensor, want: tuple[torch.Tensor, torch.Tensor], what: str = "") -> None:
    value, bound = want
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(value.shape)}"
    off = (got.detach().cpu().double() - value).abs()
    assert bool(torch.isfinite(off).all()), f"{what}: not finite"
    worst = (off / bound.clamp_min(torch.finfo(torch.float64).tiny)).max() if off.numel() else 0.0
    assert bool((off <= bound).all()), f"{what}: {float(worst):.3g} times the bound"


def residual_rmsnorm(hidden, residual, weight, eps, dtype, stream, scaled=False):
    s = hidden.double() if residual is None else hidden.double() + residual.double()
    d = s.shape[-1]
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()
    # the addition U; the mean 42 additions of 2U halved by the root, its division and the reciprocal root 3U; two products
    rel = (1 + 42 + 3 + 2) * U
    s_out = stored(s, U * s.abs(), stream)
    if not scaled:
        return stored(y, rel * y.abs(), dtype), s_out
    most = y.abs().amax(-1)
    scales = torch.where(most == 0, torch.ones_like(most), most / 448.0)
    q = y / scales[..., None]
    # e4m3: half a step is 2^-4 of the value, 2^-10 below its normal numbers; the quotient has the errors of y, of the scale and two more
    return (q, (2 * rel + 4 * U) * 448.0 + 2.0 ** -4 * q.abs() + 2.0 ** -10), (scales, (rel + 2 * U) * scales), s_out


def residual_rmsnorm_pullback(g_normed, s, weight, eps, g_residual, dtype, stream):
    s, g, w = s.double(), g_normed.double(), weight.double()
    d = s.shape[-1]
    more = torch.zeros_like(s) if g_residual is None else g_residual.double()
    inv = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)
    unit, p = s * inv, g * w
    total = inv * (p - unit * (unit * p).mean(-1, keepdim=True)) + more
    # each factor as above; the mean of products, which may cancel, goes by its magnitudes
    size = inv * (p.abs() + unit.abs() * (unit * p).abs().mean(-1, keepdim=True)) + more.abs()
    error = (3 * 48 + 42 * 2 + 8) * U * size
    rows = s.numel() // d
    terms = (g * unit).reshape(-1, d)
    # a slab is at most rows / 512 + 4 rows, the fold 64 parts of rows / 64 / 4 slabs at most and six levels
    chain = rows / 512 + 4 + min(512, rows) / 64 + 12
    g_weight = (terms.sum(0), (chain * 2 + 50) * U * terms.abs().sum(0) + 1e-45)
    return stored(total, error, dtype), stored(total, error, stream), g_weight


def _product(a, a_error, b, bias=None):
    """``a b^T`` in fp32 from an ``a`` with errors."""
    value, size, error = a @ b.t(), a.abs() @ b.abs().t(), a_error @ b.abs().t()
    if bias is not None:
        value, size = value + bias, size + bias.abs()
    return value, error + (a.shape[1] + 2) * 2 * U * size


def gated_mlp(x, fc1, fc2, fc1_bias, fc2_bias, dtype):
    x, fc1, fc2 = x.double(), fc1.double(), fc2.double()
    b1, b2 = (None if b is None else b.double() for b in (fc1_bias, fc2_bias))
    z, dz = _product(x, torch.zeros_like(x), fc1, b1)
    up, gate = z.chunk(2, -1)
    d_up, d_gate = dz.chunk(2, -1)
    silu = gate * torch.sigmoid(gate)
    a = up * silu
    # |silu'| < 1.1; exp and the division that make the sigmoid: (|gate| + 4) 2U
    da = silu.abs() * d_up + 1.1 * (up.abs() + d_up) * d_gate + (gate.abs() + 6) * 2 * U * a.abs()
    a, da = stored(a, da, dtype)
    out, d_out = _product(a, da, fc2, b2)
    return stored(out, d_out, dtype), stored(z, dz, dtype), (a, da)


def gated_mlp_vjp(g_out, x, fc1_output, down_input, fc1, fc2, dtype):
    g_out, x, z, a, fc1, fc2 = (t.double() for t in (g_out, x, fc1_output, down_input, fc1, fc2))
    up, gate = z.chunk(2, -1)
    g_a, d_a = _product(g_out, torch.zeros_like(g_out), fc2.t())
    s = torch.sigmoid(gate)
    silu, slope = gate * s, s * (1 + gate * (1 - s))
    fine = (gate.abs() + 8) * 2 * U
    g_up = stored(g_a * silu, silu.abs() * d_a + fine * (g_a * silu).abs(), dtype)
    g_gate = stored(g_a * up * slope, (up * slope).abs() * d_a + fine * (g_a * up * s).abs() * (1 + gate.abs()), dtype)
    g_z, d_z = torch.cat((g_up[0], g_gate[0]), -1), torch.cat((g_up[1], g_gate[1]), -1)
    rows = x.shape[0]
    zero = torch.zeros_like
    results = [_product(g_z, d_z, fc1.t()), _product(g_z.t(), d_z.t(), x.t()), _product(g_out.t(), zero(g_out.t()), a.t()),
               (g_z.sum(0), d_z.sum(0) + rows * 2 * U * g_z.abs().sum(0)), (g_out.sum(0), rows * 2 * U * g_out.abs().sum(0))]
    return [stored(value, error, dtype) for value, error in results]


def clip(grads, max_norm):
    """``(norm, results)``, each with its bound."""
    norm = torch.sqrt(sum((g.double().square().sum() for g in grads), torch.zeros((), dtype=torch.float64)))
    factor = min(1.0, max_norm / (float(norm) + 1e-6))
    results = [stored(g.double() * factor, 3 * U * (g.double() * factor).abs(), g.dtype) for g in grads]
    return (norm, 2 * U * norm), results
