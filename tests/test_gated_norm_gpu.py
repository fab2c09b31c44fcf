"""The norms behind and before a block with its gate and residual scale, on the GPU against their formulas in 64 bits.

Everything is fp32 between load and store: a result is off by half a step u of its type, and by half an fp32 step for each operation before, against
magnitudes that no cancellation lowers."""
from __future__ import annotations

import pytest
import torch

from latent_bounded_interfaces_amd.hip.transformer.block import gated_residual_rmsnorm, gated_residual_rmsnorm_pullback, residual_rmsnorm
from oracle import mixer_half as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS, STEP32 = 1e-5, 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(gen, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype)


def gate_of(gen, kind, shape, dtype):
    if kind is None:
        return None
    return rand(gen, *{"channel": shape[-1:], "sequence": (shape[0], *[1] * (len(shape) - 2), shape[-1]), "position": shape}[kind], dtype=dtype, std=0.7)


def close(got, want, tol, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    if got.numel():
        assert ((got - want).abs() - tol).max() <= 0, (what, float(((got - want).abs() - tol).max()), float((got - want).abs().max()))


def lowest(dtype):
    return 2.0 ** -25 if dtype == F16 else 0.0  # half precision's steps do not shrink below 2^-14


def make(gen, shape, dtype, stream, kind, weights):
    branch, residual = rand(gen, *shape, dtype=dtype), rand(gen, *shape, dtype=stream, std=2.0)
    post, weight = (rand(gen, shape[-1], dtype=weights, std=0.2, mean=1.0) for _ in range(2))
    return branch, residual, post, weight, gate_of(gen, kind, shape, dtype)


SHAPES = [(1, 1, 64), (2, 3, 8), (3, 5, 768), (2, 7, 130), (1, 4, 1), (2, 2, 1000), (1, 3, 1536), (3, 2, 2048), (1, 2, 2050), (2, 2, 5000), (1, 2, 8192), (1, 2, 9001),
          (2, 1, 16384), (4, 300, 192), (5, 13, 96)]
TYPES = [(BF16, F32, BF16), (BF16, BF16, F32), (F16, F16, F16), (F16, F32, F32), (F32, F32, F32)]


@pytest.mark.parametrize("kind", [None, "channel", "sequence", "position"])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_pullback(device, shape, types, kind):
    dtype, stream, weights = types
    gen = torch.Generator().manual_seed(31)
    branch, residual, post, weight, gate = make(gen, shape, dtype, stream, kind, weights)
    alpha, width = 0.8125, shape[-1]
    moved = [None if t is None else t.to(device) for t in (branch, residual, post, weight, gate)]
    normed, total = gated_residual_rmsnorm(*moved[:4], EPS, gate=moved[4], residual_scale=alpha)
    args = [None if t is None else t.double() for t in (branch, residual, post, weight, gate)]
    want, stream_want = oracle.gated_residual_rmsnorm(*args[:4], EPS, gate=args[4], residual_scale=alpha)
    assert normed.dtype == dtype and total.dtype == stream
    # of the sums of squares (width additions, halved by the root), the roots, divisions and products
    ops = (width / 2 + 16) * STEP32
    size = alpha * args[1].abs() + (stream_want - alpha * args[1]).abs()
    root = (stream_want.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    close(total, stream_want, half_step(stream) * stream_want.abs() + ops * size + lowest(stream), "s")
    # the norm of a sum whose elements are off by ops * size: each by its own, and all by the root's share
    spread = ((ops * size).pow(2).mean(-1, keepdim=True)).sqrt() / root
    close(normed, want, half_step(dtype) * want.abs() + ops * size / root * args[3].abs() + (ops + spread) * want.abs() + lowest(dtype), "y")

    g_normed, g_residual = rand(gen, *shape, dtype=dtype), rand(gen, *shape, dtype=stream, std=0.5)
    for more in (g_residual, None):
        got = gated_residual_rmsnorm_pullback(g_normed.to(device), moved[0], total, *moved[2:4], EPS, gate=moved[4], residual_scale=alpha,
                                              g_residual=None if more is None else more.to(device))
        wanted, sizes = pullback(g_normed, branch, total.cpu(), post, weight, gate, more, alpha)
        assert [None if t is None else t.dtype for t in got] == [dtype, stream, None if gate is None else dtype if gate.shape == branch.shape else F32, F32, F32]
        for name, a, b, c in zip(("g_branch", "g_residual", "g_gate", "g_post", "g_weight"), got, wanted, sizes):
            if b is None:
                assert a is None
                continue
            rows = branch.numel() // width if a.dtype == F32 and b.shape != branch.shape else 0
            close(a, b, half_step(a.dtype) * b.abs() + ((width + 32) + rows) * STEP32 * c + lowest(a.dtype), name)


def pullback(g_normed, branch, total, post, weight, gate, g_residual, alpha):
    """The formulas in 64 bits, and the same with every term's magnitude."""
    results = []
    for magnitude in (False, True):
        m = (lambda t: t.abs()) if magnitude else (lambda t: t)
        g, b, x, w1, w2 = (m(t.double()) for t in (g_normed, branch, total, post, weight))
        k = torch.ones((), dtype=torch.float64) if gate is None else m(gate.double())
        inv = 1 / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        inv1 = 1 / (b.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        sign = 1 if magnitude else -1
        g_s = inv * (g * w2 + sign * x * inv * (x * inv * g * w2).mean(-1, keepdim=True))
        if g_residual is not None:
            g_s = g_s + m(g_residual.double())
        unit, pulled = b * inv1, g_s * k * w1
        g_branch = inv1 * (pulled + sign * unit * (unit * pulled).mean(-1, keepdim=True))
        through = g_s * w1 * unit
        g_gate = None
        if gate is not None:
            g_gate = through if gate.shape == branch.shape else through.sum(tuple(range(branch.dim() - 1))) if gate.dim() == 1 else \
                through.sum(tuple(range(1, branch.dim() - 1)), keepdim=True)
        outer = tuple(range(branch.dim() - 1))
        results.append((g_branch, alpha * g_s, g_gate, (g_s * k * unit).sum(outer), (g * x * inv).sum(outer)))
    return results


def test_the_formulas_are_the_derivatives():
    """Of the oracle, on the CPU: what the kernels are held to is what autograd says."""
    gen = torch.Generator().manual_seed(32)
    for kind in (None, "channel", "sequence", "position"):
        branch, residual, post, weight, gate = (None if t is None else t.double().requires_grad_() for t in make(gen, (3, 4, 10), F32, F32, kind, F32))
        normed, total = oracle.gated_residual_rmsnorm(branch, residual, post, weight, EPS, gate=gate, residual_scale=0.6)
        g, g_r = rand(gen, 3, 4, 10).double(), rand(gen, 3, 4, 10).double()
        leaves = [t for t in (branch, residual, gate, post, weight) if t is not None]
        want = torch.autograd.grad((normed * g).sum() + (total * g_r).sum(), leaves)
        got = [t for t in pullback(*(None if t is None else t.detach() for t in (g, branch, total, post, weight, gate, g_r)), 0.6)[0] if t is not None]
        for a, b in zip(got, want):
            assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)


def test_without_gate_and_scale_the_second_norm_is_the_plain_one(device):
    gen = torch.Generator().manual_seed(33)
    branch, residual, post, weight, _ = (None if t is None else t.to(device) for t in make(gen, (4, 9, 768), BF16, F32, None, BF16))
    normed, total = gated_residual_rmsnorm(branch, residual, post, weight, EPS)
    again, same = residual_rmsnorm(torch.zeros_like(branch), total, weight, EPS)
    assert torch.equal(same, total) and torch.equal(again, normed)


@pytest.mark.parametrize("shape", [(0, 3, 64), (2, 0, 64), (0, 64)])
@pytest.mark.parametrize("kind", [None, "channel", "position"])
def test_no_rows(device, shape, kind):
    gen = torch.Generator().manual_seed(34)
    branch, residual, post, weight, gate = (None if t is None else t.to(device) for t in make(gen, shape, BF16, F32, kind, BF16))
    normed, total = gated_residual_rmsnorm(branch, residual, post, weight, EPS, gate=gate)
    got = gated_residual_rmsnorm_pullback(normed, branch, total, post, weight, EPS, gate=gate)
    assert normed.shape == total.shape == got[0].shape == got[1].shape == torch.Size(shape)
    assert got[3].shape == got[4].shape == (64,) and (got[3] == 0).all() and (got[4] == 0).all()
    if kind == "channel":
        assert got[2].dtype == F32 and got[2].shape == (64,) and (got[2] == 0).all()


def test_one_row_of_zeros_and_strides(device):
    gen = torch.Generator().manual_seed(35)
    branch, residual, post, weight, gate = (t.to(device) for t in make(gen, (2, 4, 96), F16, F16, "sequence", F16))
    branch[1, 2] = 0
    residual[1, 2] = 0
    want = gated_residual_rmsnorm(branch, residual, post, weight, EPS, gate=gate)
    assert (want[0][1, 2] == 0).all() and (want[1][1, 2] == 0).all()
    g = rand(gen, 2, 4, 96, dtype=F16).to(device)
    grads = gated_residual_rmsnorm_pullback(g, branch, want[1], post, weight, EPS, gate=gate)
    # Both roots of a row of zeros are eps^(-1/2) = 316, so its g_branch is gate w1 w2 g 10^5 about: past half precision's 65504 where that factor is, and
    # infinite there as any value of that size is.
    exact = pullback(*(t.cpu() for t in (g, branch, want[1], post, weight, gate)), None, 1.0)[0]
    for a, b in zip(grads, exact):
        fits = b.abs() < 65504 * (1 - 2.0 ** -10)
        assert torch.isfinite(a.cpu()[fits]).all() and (fits.all() or b is exact[0])
    assert (exact[0][1, 2].abs() > 65536).any() and torch.isinf(grads[0][1, 2]).any() and not any(torch.isnan(t).any() for t in grads)
    odd = lambda t: torch.nn.functional.pad(t.transpose(0, 1), (1, 0))[..., 1:].transpose(0, 1)  # noqa: E731
    for a, b in zip(gated_residual_rmsnorm(odd(branch), odd(residual), post, weight, EPS, gate=gate.expand(2, 1, 96)), want):
        assert torch.equal(a, b)


def test_many_gates_of_few_rows(device):
    """More gates than a launch numbers in its second dimension."""
    gen = torch.Generator().manual_seed(36)
    bsz = 65536 + 9
    branch, residual, post, weight, gate = (t.to(device) for t in make(gen, (bsz, 2, 8), F32, F32, "sequence", F32))
    _, total = gated_residual_rmsnorm(branch, residual, post, weight, EPS, gate=gate)
    g = rand(gen, bsz, 2, 8).to(device)
    got = gated_residual_rmsnorm_pullback(g, branch, total, post, weight, EPS, gate=gate)
    for rows in (slice(0, 4), slice(bsz - 4, bsz), slice(65530, 65540)):
        some = gated_residual_rmsnorm_pullback(g[rows], branch[rows], total[rows], post, weight, EPS, gate=gate[rows])
        for a, b in zip(got[:3], some[:3]):
            assert torch.equal(a[rows], b)


def test_captured_and_replayed(device):
    gen = torch.Generator().manual_seed(37)
    branch, residual, post, weight, gate = (t.to(device) for t in make(gen, (3, 50, 768), BF16, F32, "sequence", BF16))
    g = rand(gen, 3, 50, 768, dtype=BF16).to(device)

    def run(b, r):
        normed, total = gated_residual_rmsnorm(b, r, post, weight, EPS, gate=gate, residual_scale=0.5)
        return (normed, total, *gated_residual_rmsnorm_pullback(g, b, total, post, weight, EPS, gate=gate, residual_scale=0.5, g_residual=r))

    b, r = branch.clone(), residual.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(b, r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = run(b, r)
    for turn in range(4):
        b.copy_(branch.roll(turn, 1)), r.copy_(residual * (turn + 1))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(results, run(b, r)):
            assert torch.equal(got, want), turn


@pytest.mark.parametrize("shape, kind", [((3, 500, 770), "sequence"), ((3, 500, 768), "channel"), ((3, 400, 2056), "sequence"), ((2, 500, 2500), None),
                                         ((1, 600, 4104), "channel"), ((2, 300, 8191), "position"), ((1, 300, 9000), "sequence")])
@pytest.mark.parametrize("types", [(BF16, F32, BF16), (F16, F16, F16), (F32, F32, F32)])
def test_several_rows_for_each_workgroup(device, shape, types, kind):
    test_forward_and_pullback(device, shape, types, kind)
