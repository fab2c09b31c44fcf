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


@pytest.mark.parametrize("dtype,stream", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 5), (70, 64), (33, 100), (70, 768), (9, 1030), (5, 4100), (3, 12000), (5000, 200)])
def test_norm_results_in_the_place_of_inputs(rows, dim, dtype, stream, device):
    """What the C interface allows of results that are inputs: the bits of those that lie apart."""
    from latent_bounded_interfaces_amd import _lib

    lib, on = _lib.load(), torch.cuda.current_stream().cuda_stream
    gen = torch.Generator().manual_seed(rows + dim)
    h, g = (_randn(gen, rows, dim).to(dtype).to(device) for _ in range(2))
    r, gr = (_randn(gen, rows, dim).to(stream).to(device) for _ in range(2))
    w = torch.ones(dim, device=device, dtype=dtype)
    codes = [_lib.dtype_code(t) for t in (dtype, stream, dtype)]
    one = dtype == stream

    def forward(hidden, residual, normed, out):
        assert lib.lbi_residual_rmsnorm(hidden.data_ptr(), residual.data_ptr(), w.data_ptr(), normed.data_ptr(), out.data_ptr(), None, rows, dim, EPS,
                                        *codes, on) == 0
        return normed, out

    want = forward(h, r, torch.empty_like(h), torch.empty_like(r))
    for normed, out in (("h", None), (None, "r"), ("h", "r")) + ((("r", None), (None, "h"), ("r", "h")) if one else ()):
        at = {"h": h.clone(), "r": r.clone()}
        got = forward(at["h"], at["r"], at[normed] if normed else torch.empty_like(h), at[out] if out else torch.empty_like(r))
        for a, b in zip(got, want):
            assert torch.equal(a, b), (normed, out)

    need = lib.lbi_residual_rmsnorm_pullback_workspace_bytes(rows, dim)
    workspace = torch.empty(need, device=device, dtype=torch.uint8)

    def pullback(g_normed, s, more, g_hidden, g_residual):
        g_weight = torch.empty(dim, device=device)
        assert lib.lbi_residual_rmsnorm_pullback(g_normed.data_ptr(), s.data_ptr(), more.data_ptr(), w.data_ptr(), g_hidden.data_ptr(),
                                                 g_residual.data_ptr(), g_weight.data_ptr(), workspace.data_ptr(), need, rows, dim, EPS, *codes, on) == 0
        return g_hidden, g_residual, g_weight

    want = pullback(g, r, gr, torch.empty_like(h), torch.empty_like(r))
    for hidden, residual in (("g", None), (None, "gr"), ("g", "gr"), (None, "r"), ("g", "r")) + ((("gr", "g"), ("r", "gr"), ("g", "g")) if one else ()):
        at = {"g": g.clone(), "r": r.clone(), "gr": gr.clone()}
        got = pullback(at["g"], at["r"], at["gr"], at[hidden] if hidden else torch.empty_like(h), at[residual] if residual else torch.empty_like(r))
        for a, b in zip(got, want):
            assert torch.equal(a, b), (hidden, residual)


def _half_calls(device):
    """(name, call of a list of tensors, the tensors) of each function."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp, residual_rmsnorm, residual_rmsnorm_pullback

    gen = torch.Generator().manual_seed(12)
    rand = lambda *shape: _randn(gen, *shape).to(BF16).to(device)
    norm = [rand(4, 16), rand(4, 16), rand(16)]
    pullback = [*norm, rand(4, 16)]
    mlp = [rand(4, 16), rand(48, 16), rand(8, 24), rand(48), rand(8)]
    vjp = [rand(4, 8), rand(4, 16), rand(4, 48), rand(4, 24), rand(48, 16), rand(8, 24)]
    return [("residual_rmsnorm", lambda t: residual_rmsnorm(*t, EPS), norm),
            ("residual_rmsnorm_pullback", lambda t: residual_rmsnorm_pullback(*t[:3], EPS, g_residual=t[3]), pullback),
            ("gated_mlp", lambda t: gated_mlp(*t), mlp), ("gated_mlp_vjp", lambda t: gated_mlp_vjp(*t), vjp)]


@pytest.mark.filterwarnings("ignore::DeprecationWarning")  # torch's own, where it first makes a tensor with a tangent
def test_derivatives_that_would_be_lost_are_refused(device):
    """Each tensor of each function in turn: one that requires grad, and one with a tangent."""
    import torch.autograd.forward_ad as forward_ad

    for name, call, tensors in _half_calls(device):
        want = call(tensors)
        want = want if isinstance(want, tuple) else (want,)
        for i, t in enumerate(tensors):
            leaf = [*tensors[:i], t.clone().requires_grad_(), *tensors[i + 1:]]
            with pytest.raises(RuntimeError, match=f"{name} records no autograd graph"):
                call(leaf)
            with torch.no_grad():
                got = call(leaf)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want):
                assert torch.equal(a, b) and not a.requires_grad
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match=f"{name} records no autograd graph"):
                call([*tensors[:i], forward_ad.make_dual(t, torch.ones_like(t)), *tensors[i + 1:]])
        with forward_ad.dual_level():
            call(tensors)  # no tangent among them


#: (rows, D, hidden, width), hidden no multiple of 8: the products of few rows (sums of one, two and four waves), tiles, sums in parts
PADDED = [(1, 8, 7, 8), (2, 1600, 13, 40), (3, 2500, 9, 24), (70, 64, 33, 40), (67, 2048, 13, 40), (600, 40, 521, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim,hidden,width", PADDED)
def test_mlp_infinities_next_to_padding(rows, dim, hidden, width, dtype, device):
    """Columns that pad ``hidden`` take no part: a row with an infinity has the infinities and NaN that the formula gives it, its neighbours
    are as without it."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    gen = torch.Generator().manual_seed(hidden)
    x, g_out = _randn(gen, rows, dim).to(dtype), _randn(gen, rows, width).to(dtype)
    fc1, fc2 = (_randn(gen, 2 * hidden, dim).abs() + 0.5).to(dtype) / dim, (_randn(gen, width, hidden).abs() + 0.5).to(dtype) / hidden
    fc2[width // 2:] *= -1
    plain = gated_mlp(x.to(device), fc1.to(device), fc2.to(device), keep=True)
    z, a = plain[1:]
    grad = gated_mlp_vjp(g_out.to(device), x.to(device), z, a, fc1.to(device), fc2.to(device))[0]
    bad_x, bad_g = x.clone(), g_out.clone()
    bad_x[rows - 1, dim // 2], bad_g[rows - 1, 0] = float("inf"), float("inf")
    # in 64 bits, for what is finite and what is not
    up, gate = (bad_x.double() @ fc1.double().t()).chunk(2, -1)
    want_out = (up * gate * torch.sigmoid(gate)) @ fc2.double().t()
    up, gate = z.cpu().double().chunk(2, -1)
    s, g_a = torch.sigmoid(gate), bad_g.double() @ fc2.double()
    want_grad = torch.cat((g_a * gate * s, g_a * up * (s * (1 + gate * (1 - s)))), -1) @ fc1.double()
    got_out = gated_mlp(bad_x.to(device), fc1.to(device), fc2.to(device))
    got_grad = gated_mlp_vjp(bad_g.to(device), x.to(device), z, a, fc1.to(device), fc2.to(device))[0]
    assert bool(torch.isinf(want_out[-1]).all())
    for got, want, before in ((got_out, want_out, plain[0]), (got_grad, want_grad, grad)):
        assert torch.equal(got[:-1], before[:-1])
        last = got[-1].cpu().double()
        assert torch.equal(torch.isnan(last), torch.isnan(want[-1])) and torch.equal(last[torch.isinf(want[-1])], want[-1][torch.isinf(want[-1])])
        assert bool(torch.isfinite(last[torch.isfinite(want[-1])]).all())


def test_the_region_pullback_reads_what_the_forward_functions_return(device):
    """A region's cache with its MLP halves as these functions compute them, from the modules' own parameters.  Beside the reference's modules, which round
    the normalised value before its weight, the activation before its product: at most eight half steps of bf16 a layer between what is read, and
    pullbacks whose derivative in it is of order one."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, residual_rmsnorm
    from latent_bounded_interfaces_amd.hip.transformer.region import region_input_pullback_basis, region_parameter_vjp
    from oracle import transformer_region as oreg

    layers, dim = 2, 96
    backend = oreg.make_backend(dim=dim, n_heads=4, n_kv_heads=2, hidden=136, layers=layers, d_conv=4, dtype=BF16, seed=3).to(device)
    gen = torch.Generator().manual_seed(14)
    basis = _randn(gen, 2, 3, 40, dim).to(BF16).to(device)
    with torch.no_grad():
        out, cache = backend.forward_region(region_input=_randn(gen, 2, 40, dim).to(BF16).to(device), region_index=0)
        want = [region_input_pullback_basis(backend, cache, basis), *region_parameter_vjp(backend, cache, basis[:, 0]).items()]
        for block, layer in zip(backend.backbone.blocks, cache.layer_caches):
            half = layer.mlp
            half.norm_output, half.norm_input = residual_rmsnorm(layer.attention.out_proj_output, layer.attention.norm_input.float(), block.norm2.weight,
                                                                 block.norm2.eps)
            down, half.fc1_output, half.down_input = gated_mlp(half.norm_output, block.mlp.fc1.weight, block.mlp.fc2.weight, keep=True)
            assert float((down - half.down_output).float().norm() / down.float().norm()) <= 8 * 2.0 ** -8
        got = [region_input_pullback_basis(backend, cache, basis), *region_parameter_vjp(backend, cache, basis[:, 0]).items()]
    assert len(got) == len(want) > 10
    for a, b in zip(got, want):
        a, b, name = (a, b, "input") if torch.is_tensor(a) else (a[1], b[1], a[0])
        assert float((a - b).float().norm() / b.float().norm()) <= layers * 8 * 2.0 ** -8, name
