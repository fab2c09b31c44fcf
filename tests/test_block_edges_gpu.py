"""Calls of the MLP half of a block beside those of its own tests, against 64 bits with bounds by arithmetic (oracle/mlp_half.py)."""
from __future__ import annotations

import pytest
import torch

from oracle import mlp_half as truth

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-5


def _randn(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen) * std


@pytest.mark.parametrize("branch,residual_type,stream", [(BF16, F32, BF16), (F16, F32, F16), (F16, BF16, F16), (BF16, F16, BF16), (BF16, F16, F32),
                                                         (BF16, BF16, F32), (F32, BF16, F32)])
@pytest.mark.parametrize("scaled", [False, True])
def test_norm_of_a_residual_in_another_type_than_the_stream(branch, residual_type, stream, scaled, device):
    """The sum sees the residual as it is, whatever type its own is stored in."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    gen = torch.Generator().manual_seed(7)
    for rows, dim in ((33, 256), (5, 771)):
        hidden, weight = _randn(gen, rows, dim).to(branch), (1 + _randn(gen, dim, std=0.1)).to(branch)
        # next to the negative of the other summand: the digits behind its type's last are what is left
        residual = (_randn(gen, rows, dim, std=0.01) - hidden.float()).to(residual_type)
        got = residual_rmsnorm(hidden.to(device), residual.to(device), weight.to(device), EPS, residual_dtype=stream, scaled=scaled)
        assert got[0].dtype == (torch.float8_e4m3fn if scaled else branch) and got[-1].dtype == stream
        want = truth.residual_rmsnorm(hidden, residual, weight, EPS, branch, stream, scaled=scaled)
        for one, expected in zip(got, want):
            truth.assert_near(one.float(), expected)


def test_norm_of_a_residual_past_the_streams_largest_number(device):
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    hidden, residual, weight = torch.ones(2, 96, dtype=F16), torch.full((2, 96), 7e4), torch.ones(96, dtype=F16)
    residual[1] = 5.0
    normed, total = residual_rmsnorm(hidden.to(device), residual.to(device), weight.to(device), EPS, residual_dtype=F16)
    truth.assert_near(normed, truth.residual_rmsnorm(hidden, residual, weight, EPS, F16, F32)[0])
    assert bool(torch.isinf(total[0]).all()) and bool((total[1] == 6).all())


@pytest.mark.parametrize("branch,weight_type", [(F16, BF16), (BF16, F16), (BF16, torch.float64), (F16, torch.float64)])
def test_norm_of_a_weight_in_another_type(branch, weight_type, device):
    """The weight is not rounded to the branch's type, whose largest number it may exceed."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm, residual_rmsnorm_pullback

    gen = torch.Generator().manual_seed(8)
    hidden, g = _randn(gen, 9, 130).to(branch), _randn(gen, 9, 130, std=0.1).to(branch)
    weight = (1 + _randn(gen, 130, std=0.1)).to(F16).to(weight_type)
    hidden[:, 0] = 2.0 ** -10
    weight[0] = 60000.0 if weight_type == F16 else 80000.0
    held = weight.float()  # what the kernels read
    got = residual_rmsnorm(hidden.to(device), None, weight.to(device), EPS)
    truth.assert_near(got[0], truth.residual_rmsnorm(hidden, None, held, EPS, branch, branch)[0])
    got = residual_rmsnorm_pullback(g.to(device), hidden.to(device), weight.to(device), EPS)
    for one, expected in zip(got, truth.residual_rmsnorm_pullback(g, hidden, held, EPS, None, branch, branch)):
        truth.assert_near(one, expected)


@pytest.mark.parametrize("scaled", [False, True])
def test_norm_of_more_rows_than_a_launch_has_threads_for(scaled, device):
    """Rows of up to 64 columns take eight threads each, and a launch has fewer than 2^32: 2^29 rows go in two.  A few rows again and again,
    each time with the same results."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    few = 97
    rows = few * ((1 << 29) // few + 40)
    gen = torch.Generator().manual_seed(11)
    some, weight = _randn(gen, few, 1, std=0.01).to(BF16).to(device), torch.full((1,), 1.5, device=device, dtype=BF16)
    want = residual_rmsnorm(some, some, weight, EPS, scaled=scaled)
    hidden = some.repeat(rows // few, 1)
    for a, b in zip(residual_rmsnorm(hidden, hidden, weight, EPS, scaled=scaled), want):
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
        assert bool((a.view(-1, few) == b.view(1, few)).all())
