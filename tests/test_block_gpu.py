"""The MLP half of a block on the GPU, forwards and backwards, against 64 bits with bounds by arithmetic (oracle/mlp_half.py)."""
from __future__ import annotations

import pytest
import torch

from oracle import mlp_half as truth

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]
#: (rows, D): single rows, widths either side of each kernel's, odd ones, rows that do not fill a workgroup
NORM_SIZES = [(1, 1), (1, 7), (5, 8), (3, 64), (1, 768), (257, 768), (4, 512), (6, 513), (2, 1000), (9, 1025), (3, 2049), (7, 2560), (5, 4100),
              (2, 8193), (3, 16384), (1030, 96)]
EPS = 1e-5


def _randn(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen) * std


def _norm_inputs(rows, dim, dtype, stream, seed=0):
    gen = torch.Generator().manual_seed(1000 * rows + dim + seed)
    return (_randn(gen, rows, dim).to(dtype), _randn(gen, rows, dim, std=2.0).to(stream), (1 + _randn(gen, dim, std=0.1)).to(dtype),
            _randn(gen, rows, dim, std=0.5).to(stream))


def _on(device, *tensors):
    return [None if t is None else t.to(device) for t in tensors]


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
def test_norm(rows, dim, dtype, stream, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    hidden, residual, weight, _ = _norm_inputs(rows, dim, dtype, stream)
    normed, total = residual_rmsnorm(*_on(device, hidden, residual, weight), EPS)
    assert normed.dtype == dtype and total.dtype == stream
    want = truth.residual_rmsnorm(hidden, residual, weight, EPS, dtype, stream)
    truth.assert_near(normed, want[0], "normed")
    truth.assert_near(total, want[1], "residual")


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
def test_norm_scaled(rows, dim, dtype, stream, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    hidden, residual, weight, _ = _norm_inputs(rows, dim, dtype, stream, seed=1)
    normed, scales, total = residual_rmsnorm(*_on(device, hidden, residual, weight), EPS, scaled=True)
    assert normed.dtype == torch.float8_e4m3fn and scales.dtype == F32 and scales.shape == (rows,)
    want = truth.residual_rmsnorm(hidden, residual, weight, EPS, dtype, stream, scaled=True)
    for got, one, what in zip((normed.float(), scales, total), want, ("normed", "scales", "residual")):
        truth.assert_near(got, one, what)


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
def test_norm_pullback(rows, dim, dtype, stream, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm_pullback

    g_normed, s, weight, g_residual = _norm_inputs(rows, dim, dtype, stream, seed=2)
    for extra in (g_residual, None):
        got = residual_rmsnorm_pullback(*_on(device, g_normed, s, weight), EPS, g_residual=_on(device, extra)[0])
        assert got[0].dtype == dtype and got[1].dtype == stream and got[2].dtype == F32
        want = truth.residual_rmsnorm_pullback(g_normed, s, weight, EPS, extra, dtype, stream)
        for one, expected, what in zip(got, want, ("g_hidden", "g_residual", "g_weight")):
            truth.assert_near(one, expected, what)


def test_norm_pullback_against_differences(device):
    """The pullback of fp32 against central differences of the operator's formula in 64 bits."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm_pullback

    gen = torch.Generator().manual_seed(3)
    s, weight, g = _randn(gen, 2, 12), 1 + _randn(gen, 12, std=0.1), _randn(gen, 2, 12)

    def value(s, w):
        return float((g.double() * s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * w).sum())

    got = residual_rmsnorm_pullback(*_on(device, g, s, weight), EPS)
    step = 1e-6
    for at, grad in ((0, got[1]), (1, got[2])):
        args = [s.double(), weight.double()]
        want = torch.empty(args[at].numel(), dtype=torch.float64)
        for i in range(want.numel()):
            sides = []
            for sign in (step, -step):
                moved = [a.clone() for a in args]
                moved[at].view(-1)[i] += sign
                sides.append(value(*moved))
            want[i] = (sides[0] - sides[1]) / (2 * step)
        # differences: h^2 times a third derivative of order 1, and the cancellation of values of order 10 at 2^-53 / h
        assert float((grad.cpu().double().view(-1) - want).abs().max()) <= 1e-7 + 1e-5 * float(want.abs().max())


@pytest.mark.parametrize("stream", [F32, BF16])
def test_norm_without_residual(stream, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    hidden, _, weight, _ = _norm_inputs(33, 200, BF16, stream)
    normed, total = residual_rmsnorm(*_on(device, hidden, None, weight), EPS, residual_dtype=stream)
    want = truth.residual_rmsnorm(hidden, None, weight, EPS, BF16, stream)
    truth.assert_near(normed, want[0])
    assert total.dtype == stream and torch.equal(total.cpu(), hidden.to(stream))


@pytest.mark.parametrize("dim", [768, 771])
@pytest.mark.parametrize("scaled", [False, True])
def test_norm_of_tensors_that_start_anywhere_and_lie_apart(dim, scaled, device):
    """Views at odd element offsets, strided rows, transposed storage, an fp32 weight."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm, residual_rmsnorm_pullback

    gen = torch.Generator().manual_seed(dim)
    rows = 11
    flat = _randn(gen, rows * dim + 3).to(BF16).to(device)
    hidden = flat[3:].view(rows, dim)
    residual = _randn(gen, rows, dim + 5).to(device)[:, 2:2 + dim]
    weight = (1 + _randn(gen, dim + 1, std=0.1)).to(device)[1:]
    got = residual_rmsnorm(hidden, residual, weight, EPS, scaled=scaled)
    same = residual_rmsnorm(hidden.clone(), residual.contiguous(), weight.clone(), EPS, scaled=scaled)
    for a, b in zip(got, same):
        assert torch.equal(a.float(), b.float())
    want = truth.residual_rmsnorm(hidden.cpu(), residual.cpu(), weight.cpu(), EPS, BF16, F32, scaled=scaled)
    for one, expected in zip(got, want):
        truth.assert_near(one.float(), expected)
    turned = residual.t().contiguous().t()
    for a, b in zip(residual_rmsnorm_pullback(hidden, turned, weight, EPS), residual_rmsnorm_pullback(hidden.clone(), residual, weight.clone(), EPS)):
        assert torch.equal(a, b)


def test_norm_of_special_rows(device):
    """Rows of zeros, of the smallest and largest numbers, with infinities and NaN: a row's results are its own."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm

    gen = torch.Generator().manual_seed(9)
    hidden = _randn(gen, 8, 96)
    hidden[1] = 0
    hidden[2] = 0
    hidden[2, 40] = 1e-38
    hidden[3, 5] = float("inf")
    hidden[4, 6] = float("nan")
    hidden[5] = 1e18
    hidden[6, :] = 0
    weight = torch.ones(96)
    fine = [0, 1, 2, 5, 6, 7]
    want = truth.residual_rmsnorm(hidden, None, weight, EPS, F32, F32)
    normed, total = residual_rmsnorm(*_on(device, hidden, None, weight), EPS)
    truth.assert_near(normed[fine], tuple(t[fine] for t in want[0]))
    assert torch.equal(total.cpu()[fine], hidden[fine])
    # an infinite element's own place is not a number, the others are 0; NaN spreads over its row
    assert bool(torch.isnan(normed[3, 5])) and int((normed[3] == 0).sum()) == 95 and bool(torch.isnan(normed[4]).all())
    q, scales, _ = residual_rmsnorm(*_on(device, hidden, None, weight), EPS, scaled=True)
    assert scales[1].item() == 1.0 and scales[6].item() == 1.0 and not q[1].float().any()
    scaled = (q.float() * scales[:, None]).cpu().double()
    y = want[0][0]
    for r in fine:  # half a step of e4m3 next to a row's largest magnitude, and what fp32 adds
        bound = 2.0 ** -4 * y[r].abs() + (2.0 ** -10 + 448 * 2.0 ** -17) * scales[r].cpu().double()
        assert bool(((scaled[r] - y[r]).abs() <= bound).all())
    assert bool(torch.isnan(scales[3])) and bool(torch.isnan(scales[4]))


def test_norm_of_nothing(device):
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm, residual_rmsnorm_pullback

    hidden, weight = torch.zeros(2, 0, 32, device=device), torch.ones(32, device=device)
    normed, total = residual_rmsnorm(hidden, hidden, weight, EPS)
    assert normed.shape == total.shape == hidden.shape
    assert residual_rmsnorm(hidden, None, weight, EPS, scaled=True)[1].shape == (2, 0)
    g_hidden, g_residual, g_weight = residual_rmsnorm_pullback(hidden, hidden, weight, EPS)
    assert g_hidden.shape == g_residual.shape == hidden.shape and not g_weight.any()


def _mlp_inputs(rows, dim, hidden, width, dtype, bias, seed=0):
    gen = torch.Generator().manual_seed(rows + 7 * dim + 13 * hidden + width + seed)
    x, g_out = _randn(gen, rows, dim).to(dtype), _randn(gen, rows, width).to(dtype)
    fc1, fc2 = _randn(gen, 2 * hidden, dim, std=dim ** -0.5).to(dtype), _randn(gen, width, hidden, std=hidden ** -0.5).to(dtype)
    b1, b2 = (_randn(gen, 2 * hidden, std=0.3).to(dtype), _randn(gen, width, std=0.3).to(dtype)) if bias else (None, None)
    return x, fc1, fc2, b1, b2, g_out


#: (rows, D, hidden, width): single rows, sizes that end inside tiles, widths of no whole 16-byte pieces, more rows than a tile
MLP_SIZES = [(1, 8, 8, 8), (1, 64, 128, 64), (1, 768, 512, 768), (2, 40, 24, 56), (3, 256, 320, 128), (5, 100, 72, 100), (8, 33, 17, 9), (16, 128, 192, 128),
             (17, 264, 136, 200), (31, 512, 64, 512), (64, 96, 160, 96), (77, 320, 200, 320), (129, 72, 264, 136), (200, 256, 512, 128),
             (300, 64, 64, 264), (513, 136, 72, 64), (1, 2048, 24, 2056), (700, 264, 328, 264)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim,hidden,width", MLP_SIZES)
def test_mlp(rows, dim, hidden, width, dtype, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp

    for bias in (False, True):
        args = _mlp_inputs(rows, dim, hidden, width, dtype, bias)[:5]
        out, fc1_output, down_input = gated_mlp(*_on(device, *args), keep=True)
        alone = gated_mlp(*_on(device, *args))
        assert out.dtype == fc1_output.dtype == down_input.dtype == dtype and torch.equal(out, alone)
        want = truth.gated_mlp(*args, dtype)
        for got, one, what in zip((out, fc1_output, down_input), want, ("out", "fc1_output", "down_input")):
            truth.assert_near(got, one, what)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim,hidden,width", MLP_SIZES)
def test_mlp_vjp(rows, dim, hidden, width, dtype, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp_vjp

    x, fc1, fc2, _, _, g_out = _mlp_inputs(rows, dim, hidden, width, dtype, False, seed=1)
    gen = torch.Generator().manual_seed(rows)
    fc1_output = _randn(gen, rows, 2 * hidden, std=1.5).to(dtype)
    up, gate = fc1_output.float().chunk(2, -1)
    down_input = (up * gate * torch.sigmoid(gate)).to(dtype)
    args = (g_out, x, fc1_output, down_input, fc1, fc2)
    got = gated_mlp_vjp(*_on(device, *args), bias=True)
    want = truth.gated_mlp_vjp(*args, dtype)
    for one, expected, what in zip(got, want, ("g_x", "g_fc1_weight", "g_fc2_weight", "g_fc1_bias", "g_fc2_bias")):
        assert one.dtype == dtype
        truth.assert_near(one, expected, what)
    for a, b in zip(gated_mlp_vjp(*_on(device, *args)), got):
        assert torch.equal(a, b)


#: Sizes that between them take every tile of every product of both directions, on 256 compute units, with sums whole and cut into parts
MLP_TILES = [(5632, 36, 3902, 154), (179, 2558, 2821, 87), (5886, 164, 2394, 26), (3524, 1682, 19, 340), (5461, 2377, 16, 169),
             (8245, 31, 151, 520), (1435, 172, 4013, 621), (1, 903, 2069, 34), (1, 1698, 1764, 1105), (1, 2100, 1922, 27), (2615, 21, 17, 2370),
             (1109, 17, 1982, 16), (8623, 411, 16, 69), (5548, 91, 16, 1411), (6510, 17, 23, 939), (1214, 22, 2444, 18), (8274, 697, 16, 20),
             (3889, 2182, 17, 18), (6409, 16, 965, 20), (8019, 28, 79, 1607), (6898, 29, 638, 513), (254, 1904, 4009, 653), (5, 1108, 18, 201),
             (75, 1413, 16, 371), (67, 21, 729, 25), (5, 27, 1141, 18), (7711, 34, 527, 22), (1, 164, 4011, 962), (78, 825, 3979, 2026)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim,hidden,width", MLP_TILES)
def test_mlp_tiles(rows, dim, hidden, width, dtype, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    x, fc1, fc2, b1, b2, g_out = _on(device, *_mlp_inputs(rows, dim, hidden, width, dtype, True, seed=2))
    got = gated_mlp(x, fc1, fc2, b1, b2, keep=True)
    grads = gated_mlp_vjp(g_out, x, got[1], got[2], fc1, fc2, bias=True)
    want = (*truth.gated_mlp(x, fc1, fc2, b1, b2, dtype), *truth.gated_mlp_vjp(g_out, x, got[1], got[2], fc1, fc2, dtype))
    names = ("out", "fc1_output", "down_input", "g_x", "g_fc1_weight", "g_fc2_weight", "g_fc1_bias", "g_fc2_bias")
    for one, (value, bound), what in zip((*got, *grads), want, names):
        truth.assert_near(one, (value.cpu(), bound.cpu()), what)


def test_mlp_offsets_past_32_bits(device):
    """More than 2^31 elements of fc1_output.  The cotangent is zero but for the last rows, whose weight gradients are all there is."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    rows, dim, hidden, few = 131075, 64, 8200, 64
    x, fc1, fc2, _, _, g_out = _on(device, *_mlp_inputs(rows, dim, hidden, dim, BF16, False))
    g_out[:-few] = 0
    got = gated_mlp(x, fc1, fc2, keep=True)
    for part in (slice(0, few), slice(rows - few, rows)):
        for one, (value, bound), what in zip(got, truth.gated_mlp(x[part], fc1, fc2, None, None, BF16), ("out", "fc1_output", "down_input")):
            truth.assert_near(one[part], (value.cpu(), bound.cpu()), what)
    grads = gated_mlp_vjp(g_out, x, got[1], got[2], fc1, fc2, bias=True)
    last = [t[-few:] for t in (g_out, x, got[1], got[2])]
    assert not grads[0][:-few].any()
    for one, (value, bound), what in zip((grads[0][-few:], *grads[1:]), truth.gated_mlp_vjp(*last, fc1, fc2, BF16), range(5)):
        truth.assert_near(one, (value.cpu(), bound.cpu()), str(what))


@pytest.mark.parametrize("scaled", [False, True])
def test_norm_offsets_past_32_bits(scaled, device):
    """More than 2^31 elements: a row's results do not depend on where it lies."""
    from latent_bounded_interfaces_amd.hip.transformer.block import residual_rmsnorm, residual_rmsnorm_pullback

    rows, dim, few = 131100, 16384, 40
    gen = torch.Generator().manual_seed(5)
    some, weight = _randn(gen, few, dim).to(BF16).to(device), (1 + _randn(gen, dim, std=0.1)).to(BF16).to(device)
    hidden = torch.zeros(rows, dim, device=device, dtype=BF16)
    hidden[-few:] = some
    got, want = residual_rmsnorm(hidden, None, weight, EPS, scaled=scaled), residual_rmsnorm(some, None, weight, EPS, scaled=scaled)
    for a, b in zip(got, want):
        assert torch.equal(a[-few:].float(), b.float())
    if not scaled:
        grad = residual_rmsnorm_pullback(hidden, hidden, weight, EPS, g_residual=hidden)
        alone = residual_rmsnorm_pullback(some, some, weight, EPS, g_residual=some)
        assert torch.equal(grad[0][-few:], alone[0]) and not grad[0][:-few].any()
        value, bound = truth.residual_rmsnorm_pullback(some.cpu(), some.cpu(), weight.cpu(), EPS, some.cpu(), BF16, BF16)[2]
        chain = rows / 512 + 4 + 8 + 12  # the bound's own slabs, of all rows
        truth.assert_near(grad[2], (value, bound * ((chain * 2 + 50) / 50)), "g_weight")


def test_mlp_gradients_of_the_formula(device):
    """Forward and pullback together against autograd of the formula in 64 bits: what the roundings in between add is bounded by that
    of the three 16-bit tensors on the way, 4 half steps of the largest magnitudes."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    x, fc1, fc2, b1, b2, g_out = _mlp_inputs(45, 96, 80, 72, F16, True)
    _, fc1_output, down_input = gated_mlp(*_on(device, x, fc1, fc2, b1, b2), keep=True)
    got = gated_mlp_vjp(*_on(device, g_out, x), fc1_output, down_input, *_on(device, fc1, fc2), bias=True)
    leaves = [t.double().requires_grad_() for t in (x, fc1, fc2, b1, b2)]
    up, gate = (leaves[0] @ leaves[1].t() + leaves[3]).chunk(2, -1)
    ((up * torch.nn.functional.silu(gate)) @ leaves[2].t() + leaves[4]).backward(g_out.double())
    for one, leaf in zip(got, leaves):
        off = (one.cpu().double() - leaf.grad).norm() / leaf.grad.norm()
        assert float(off) <= 4 * 2.0 ** -11


def test_mlp_of_other_layouts(device):
    """Leading dimensions, strided inputs, tensors off the 16-byte grid, fp32 parameters."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    x, fc1, fc2, b1, b2, g_out = (t.to(device) for t in _mlp_inputs(24, 64, 48, 40, BF16, True))
    want = gated_mlp(x, fc1, fc2, b1, b2, keep=True)
    grads = gated_mlp_vjp(g_out, x, want[1], want[2], fc1, fc2)
    off = torch.empty(24 * 64 + 1, device=device, dtype=BF16)[1:].view(24, 64).copy_(x)
    wide = torch.zeros(24, 100, device=device, dtype=BF16)
    wide[:, 8:72] = x
    turned = fc1.t().contiguous().t()
    for other in (off, wide[:, 8:72]):
        got = gated_mlp(other.view(2, 3, 4, 64) if other.is_contiguous() else other, turned, fc2.float(), b1.float(), b2, keep=True)
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(b.shape), b)
        for a, b in zip(gated_mlp_vjp(g_out.t().contiguous().t(), other, want[1], want[2], turned, fc2.float()), grads):
            assert torch.equal(a, b)
    cube = [t.view(4, 6, -1) for t in (g_out, x, want[1], want[2])]
    for a, b in zip(gated_mlp_vjp(*cube, fc1, fc2), grads):
        assert torch.equal(a.reshape(b.shape), b)


def test_mlp_of_nothing_and_of_values_that_are_not_finite(device):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    x, fc1, fc2, b1, b2, g_out = (t.to(device) for t in _mlp_inputs(40, 72, 136, 72, BF16, True))
    none = x[:0]
    out, fc1_output, down_input = gated_mlp(none, fc1, fc2, keep=True)
    assert out.shape == (0, 72) and fc1_output.shape == (0, 272) and down_input.shape == (0, 136)
    grads = gated_mlp_vjp(none, none, fc1_output, down_input, fc1, fc2, bias=True)
    assert grads[0].shape == (0, 72) and not any(g.any() for g in grads[1:]) and grads[1].shape == fc1.shape
    # a row's numbers stay in it: tiles are shared, sums are not
    want = gated_mlp(x, fc1, fc2, b1, b2)
    bad = x.clone()
    bad[39] = float("nan")
    bad[7, 3] = float("inf")
    got = gated_mlp(bad, fc1, fc2, b1, b2)
    rest = [r for r in range(40) if r not in (7, 39)]
    assert torch.equal(got[rest], want[rest]) and bool(torch.isnan(got[39]).all())
    # and what lies behind the weights' rows does not enter: gates far out close or open without NaN
    far = gated_mlp(x * 2e4, fc1, fc2, keep=True)
    assert bool(torch.isfinite(far[2]).all())


def test_results_repeat_and_streams(device):
    """The same bits on every run, on the current stream of the tensors' device."""
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp, residual_rmsnorm_pullback

    x, fc1, fc2, b1, b2, g_out = (t.to(device) for t in _mlp_inputs(1500, 256, 264, 256, BF16, True))

    def call():
        out, z, a = gated_mlp(x, fc1, fc2, b1, b2, keep=True)
        return (out, z, a, *gated_mlp_vjp(g_out, x, z, a, fc1, fc2, bias=True), *residual_rmsnorm_pullback(g_out, x, b2, EPS))

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def _training_half(x, residual, norm, fc1, fc2, b1, b2, g_out, g_residual):
    """The MLP half of a block, forwards and backwards, and the clipping of its gradients."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients
    from latent_bounded_interfaces_amd.hip.transformer.block import (gated_mlp, gated_mlp_vjp, residual_rmsnorm,
                                                                     residual_rmsnorm_pullback)

    normed, stream = residual_rmsnorm(x, residual, norm, EPS)
    out, z, a = gated_mlp(normed, fc1, fc2, b1, b2, keep=True)
    g_normed, *grads = gated_mlp_vjp(g_out, normed, z, a, fc1, fc2, bias=True)
    g_x, g_in, g_norm = residual_rmsnorm_pullback(g_normed, stream, norm, EPS, g_residual=g_residual)
    clipped = [torch.empty_like(g) for g in (*grads, g_norm)]
    norm_of_all = clip_gradients([*grads, g_norm], 1.0, out=clipped)
    return out, stream, g_x, g_in, norm_of_all, *clipped


def _half_inputs(gen, device, rows=130, dim=96, hidden=136):
    def rand(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=gen) * std).to(dtype).to(device)

    return [rand(rows, dim), rand(rows, dim, std=2.0, dtype=F32), 1 + rand(dim, std=0.1), rand(2 * hidden, dim, std=dim ** -0.5),
            rand(dim, hidden, std=hidden ** -0.5), rand(2 * hidden, std=0.1), rand(dim, std=0.1), rand(rows, dim), rand(rows, dim, dtype=F32)]


def test_a_training_step_of_the_half(device):
    """All of it against autograd in 64 bits.  Five tensors of bf16 lie on the longest way (normed, fc1_output, down_input, the cotangents
    of fc1_output and normed) beside the result: six half steps in the 2-norm."""
    args = _half_inputs(torch.Generator().manual_seed(4), device)
    got = _training_half(*args)
    x, residual, norm, fc1, fc2, b1, b2 = leaves = [t.cpu().double().requires_grad_() for t in args[:7]]
    stream = x + residual
    normed = stream * torch.rsqrt(stream.square().mean(-1, keepdim=True) + EPS) * norm
    up, gate = (normed @ fc1.t() + b1).chunk(2, -1)
    out = (up * torch.nn.functional.silu(gate)) @ fc2.t() + b2
    torch.autograd.backward([out, stream], [args[7].cpu().double(), args[8].cpu().double()])
    parameters = [t.grad for t in (fc1, fc2, b1, b2, norm)]
    total = torch.sqrt(sum(g.square().sum() for g in parameters))
    want = [out, stream, x.grad, residual.grad, total, *(g / (total + 1e-6) for g in parameters)]
    assert float(total) > 1
    for i, (a, b) in enumerate(zip(got, want)):
        assert float((a.cpu().double() - b.detach()).norm() / b.detach().norm()) <= 6 * 2.0 ** -8, i


def test_captured_step_replays_with_new_inputs(device):
    """Nothing allocates device memory by itself, synchronises or clears by a stream's memset; two graphs share no workspace."""
    gen = torch.Generator().manual_seed(6)
    static = _half_inputs(gen, device), _half_inputs(gen, device, rows=7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for args in static:
            _training_half(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, captured = [], []
    for args in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(_training_half(*args))
        graphs.append(graph)
    for _ in range(3):
        values = _half_inputs(gen, device), _half_inputs(gen, device, rows=7)
        for into, new in zip(static, values):
            for dst, src in zip(into, new):
                dst.copy_(src)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in results] for results in captured]
        for results, new in zip(got, values):
            for a, b in zip(results, _training_half(*new)):  # eager work between replays
                assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_refusals_on_the_device(device):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp, residual_rmsnorm, residual_rmsnorm_pullback

    x, fc1, fc2, b1, b2, g_out = (t.to(device) for t in _mlp_inputs(4, 16, 24, 32, BF16, True))
    weight = torch.ones(16, device=device, dtype=BF16)
    with pytest.raises(ValueError, match="shaped like hidden"):
        residual_rmsnorm(x, x[:2], weight, EPS)
    with pytest.raises(ValueError, match="residual stream"):
        residual_rmsnorm(x, x.half(), weight, EPS)
    with pytest.raises(ValueError, match="weight"):
        residual_rmsnorm(x, x, weight[1:], EPS)
    with pytest.raises(RuntimeError, match="no autograd graph"):
        residual_rmsnorm(x, x, weight.clone().requires_grad_(), EPS)
    with pytest.raises(RuntimeError, match="16384"):
        residual_rmsnorm(torch.zeros(1, 16385, device=device), None, torch.ones(16385, device=device), EPS)
    with pytest.raises(ValueError, match="g_residual"):
        residual_rmsnorm_pullback(x, x.float(), weight, EPS, g_residual=x)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        gated_mlp(x.float(), fc1.float(), fc2.float())
    with pytest.raises(ValueError, match="2 \\* hidden"):
        gated_mlp(x, fc1[:-2], fc2)
    with pytest.raises(ValueError, match="fc1_bias"):
        gated_mlp(x, fc1, fc2, b2, b2)
    with pytest.raises(RuntimeError, match="no autograd graph"):
        gated_mlp(x, fc1.clone().requires_grad_(), fc2)
    with torch.no_grad():
        gated_mlp(x, fc1.clone().requires_grad_(), fc2)
    z, a = gated_mlp(x, fc1, fc2, keep=True)[1:]
    with pytest.raises(ValueError, match="down_input"):
        gated_mlp_vjp(g_out, x, z, a.half(), fc1, fc2)
    with pytest.raises(ValueError, match="g_out"):
        gated_mlp_vjp(g_out[:, :-1], x, z, a, fc1, fc2)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_mlp(x.cpu(), fc1, fc2)
