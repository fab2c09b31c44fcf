"""The gated norms' pullback for more gates than one launch has workgroups for, on the GPU."""
from __future__ import annotations

import pytest
import torch

import test_gated_norm_gpu as base
from latent_bounded_interfaces_amd.hip.transformer.block import gated_residual_rmsnorm, gated_residual_rmsnorm_pullback

pytestmark = pytest.mark.gpu

EPS = 1e-5


def test_more_gates_than_a_launch_has_workgroups_for(device):
    """A gate for each two rows, 2^24 + 5 of them: a workgroup each, of 256 threads."""
    gen = torch.Generator(device=device).manual_seed(48)
    bsz, dim = 2 ** 24 + 5, 8
    branch, residual, g = (torch.randn(bsz, 2, dim, generator=gen, device=device, dtype=torch.bfloat16) for _ in range(3))
    gate = torch.randn(bsz, 1, dim, generator=gen, device=device, dtype=torch.bfloat16)
    post, weight = (1 + 0.1 * torch.randn(dim, generator=gen, device=device) for _ in range(2))
    _, total = gated_residual_rmsnorm(branch, residual, post, weight, EPS, gate=gate)
    got = gated_residual_rmsnorm_pullback(g, branch, total, post, weight, EPS, gate=gate)
    torch.cuda.synchronize()
    some = [gated_residual_rmsnorm_pullback(g[rows], branch[rows], total[rows], post, weight, EPS, gate=gate[rows])
            for rows in (slice(0, 2 ** 23), slice(2 ** 23, 2 ** 24 - 3), slice(2 ** 24 - 3, bsz))]
    torch.cuda.synchronize()
    for i in range(3):
        assert torch.equal(got[i], torch.cat([part[i] for part in some]))
    # the weights' gradients: a thread adds 2^18 of a column's shares one after the other, each of two terms, and 64 threads' sums are added in a tree, so they are off by
    # (2^18 + 16) fp32 half steps of the terms' magnitudes at most, and the terms by 40 half steps of theirs
    g_w, sizes = 0.0, 0.0
    for rows in torch.arange(bsz, device=device).split(2 ** 22):
        x = total[rows].double()
        term = g[rows].double() * x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        g_w, sizes = g_w + term.sum((0, 1)), sizes + term.abs().sum((0, 1))
    assert ((got[4].double() - g_w).abs() - (2 ** 18 + 64) * 2.0 ** -24 * sizes).max() <= 0


@pytest.mark.parametrize("dtype, stream", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("positions", [(1,), (4,), (1, 1)])
def test_a_gate_of_each_sequence_has_its_gradient_in_fp32(device, dtype, stream, positions):
    gen = torch.Generator().manual_seed(49)
    bsz, dim = 3, 776
    branch, g = (base.rand(gen, bsz, *positions, dim, dtype=dtype) for _ in range(2))
    residual = base.rand(gen, bsz, *positions, dim, dtype=stream)
    gate = base.rand(gen, bsz, *[1] * len(positions), dim, dtype=dtype)
    post, weight = (base.rand(gen, dim, std=0.2, mean=1.0) for _ in range(2))
    moved = [t.to(device) for t in (branch, residual, post, weight, gate)]
    _, total = gated_residual_rmsnorm(*moved[:4], EPS, gate=moved[4])
    got = gated_residual_rmsnorm_pullback(g.to(device), moved[0], total, *moved[2:4], EPS, gate=moved[4], sequence_gate=True)
    assert [t.dtype for t in got] == [dtype, stream, torch.float32, torch.float32, torch.float32] and got[2].shape == gate.shape
    wanted, sizes = base.pullback(g, branch, total.cpu(), post, weight, gate, None, 1.0)
    for name, a, b, c in zip(("g_branch", "g_residual", "g_gate", "g_post", "g_weight"), got, wanted, sizes):
        base.close(a, b, base.half_step(a.dtype) * b.abs() + (dim + 32 + bsz * 4) * base.STEP32 * c + base.lowest(a.dtype), name)
    # the same numbers as those of a gate of each position, before their rounding
    if positions != (4,):
        each = gated_residual_rmsnorm_pullback(g.to(device), moved[0], total, *moved[2:4], EPS, gate=moved[4])
        assert each[2].dtype == dtype and torch.equal(got[2].to(dtype), each[2])
