"""Clipping by the global norm on the GPU, against 64 bits with bounds by arithmetic (oracle/mlp_half.py)."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import mlp_half as truth

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _grads(counts, dtypes, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(counts)]


@pytest.mark.parametrize("dtypes", [(F32,), (BF16, F32), (F16, BF16, F32)])
@pytest.mark.parametrize("counts", [(1,), (7, 0, 8), (1, 2, 3, 4, 5), (8192,), (8191, 8193), (100003, 1, 65536), (40,) * 99, (33,) * 100, (17,) * 101,
                                    (2049, 5) * 130, (9_000_000, 3)])
@pytest.mark.parametrize("max_norm", [0.5, math.inf])
def test_clip(counts, dtypes, max_norm, device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients, gradient_norm

    grads = _grads(counts, dtypes, seed=len(counts))
    on = [g.to(device) for g in grads]
    want_norm, want = truth.clip(grads, max_norm)
    outs = [torch.full_like(g, float("nan")) for g in on]
    norm = clip_gradients(on, max_norm, out=outs)
    assert norm.dtype == F32 and norm.shape == () and norm.device == on[0].device
    truth.assert_near(norm, want_norm)
    assert torch.equal(gradient_norm(on), norm)
    for got, one, before, now in zip(outs, want, grads, on):
        truth.assert_near(got, one)
        assert torch.equal(before, now.cpu())
    again = clip_gradients(on, max_norm)  # in place
    assert torch.equal(again, norm)
    for a, b in zip(on, outs):
        assert torch.equal(a, b)


def test_below_the_limit_nothing_changes(device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    grads = [g.to(device) for g in _grads((1000, 77), (BF16, F32), std=1e-3)]
    before = [g.clone() for g in grads]
    outs = [torch.empty_like(g) for g in grads]
    clip_gradients(grads, 1.0, out=outs)
    clip_gradients(grads, 1.0)
    for a, b, c in zip(grads, before, outs):
        assert torch.equal(a, b) and torch.equal(c, b)


def test_largest_and_smallest_numbers(device):
    """Squares of fp32 neither overflow nor vanish."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    for std in (1e30, 1e-30):
        grads = _grads((5000,), (F32,), std=std)
        want_norm, want = truth.clip(grads, std)
        on = [g.to(device) for g in grads]
        truth.assert_near(clip_gradients(on, std), want_norm)
        truth.assert_near(on[0], want[0])


def test_values_that_are_not_finite(device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    for bad in (float("nan"), float("inf")):
        grads = [g.to(device) for g in _grads((500, 20), (F32, BF16))]
        grads[1][3] = bad
        norm = clip_gradients(grads, 1.0)
        reference = [g.clone().float() for g in grads]
        if math.isnan(bad):
            assert bool(torch.isnan(norm)) and all(bool(torch.isnan(g).all()) for g in reference)
        else:
            assert math.isinf(norm.item()) and not reference[0].any() and bool(torch.isnan(reference[1][3]))
            assert int((reference[1] == 0).sum()) == 19


def test_more_elements_than_32_bits_count(device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    count = 2 ** 31 + 5
    grads = [torch.full((count,), 0.5, device=device, dtype=torch.bfloat16), torch.full((3,), 2.0, device=device)]
    total = (count * 0.25 + 12.0) ** 0.5
    norm = clip_gradients(grads, total / 4)
    assert abs(float(norm) - total) <= 2 * 2.0 ** -24 * total
    # a quarter of 0.5 and 2 exactly, but for the factor's own 1e-6 / norm and its rounding, which bf16 rounds away
    assert bool((grads[0] == 0.125).all()) and bool(((grads[1] - 0.5).abs() <= 2.0 ** -22).all())


def test_layouts(device):
    """Tensors off the vector grid, transposed, strided, expanded; one of them twice."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    gen = torch.Generator().manual_seed(2)
    flat = torch.randn(100_003, generator=gen).to(BF16).to(device)
    base = torch.randn(64, 96, generator=gen).to(device)
    grads = [flat[1:50_002], flat[50_002:], base.t(), torch.randn(40, 50, generator=gen).to(device)[:, 3:20], torch.randn(30, 1, generator=gen).to(device).expand(30, 7)]
    want_norm, want = truth.clip([g.cpu() for g in grads], 2.0)
    outs = [torch.empty_like(g) for g in grads[:3]] + [torch.empty(40, 60, device=device)[:, 5:22], torch.empty(30, 7, device=device)]
    truth.assert_near(clip_gradients(grads, 2.0, out=outs), want_norm)
    for got, one in zip(outs, want):
        truth.assert_near(got, one)
    crossed = [torch.empty(64, 96, device=device).t()]  # contiguous input, result lying otherwise
    clip_gradients([base.t().contiguous()], 0.25, out=crossed)
    truth.assert_near(crossed[0], truth.clip([base.t().cpu()], 0.25)[1][0])
    clip_gradients(grads[:4], 2.0)  # in place
    want_norm, want = truth.clip([g.cpu() for g in (flat[1:],)], 2.0)
    twice = [torch.empty_like(base), torch.empty_like(base)]
    before = base.clone()
    want_norm, want = truth.clip([before.cpu(), before.cpu()], 1.0)
    truth.assert_near(clip_gradients([base, base], 1.0, out=twice), want_norm)
    assert torch.equal(twice[0], twice[1])
    truth.assert_near(twice[0], want[0])


def test_in_place_strided(device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    base = torch.arange(1.0, 61.0).view(6, 10).to(device)
    before = base.clone().cpu()
    clip_gradients([base[:, :4], base[:, 4:]], 1.0)  # two halves of one storage
    truth.assert_near(base, truth.clip([before], 1.0)[1][0])


def test_refusals(device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients, gradient_norm

    a, b = torch.ones(64, device=device), torch.ones(64, device=device)
    with pytest.raises(RuntimeError, match="overlaps"):
        clip_gradients([a, a], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        clip_gradients([a, b], 1.0, out=[b, a])
    with pytest.raises(RuntimeError, match="overlaps"):
        clip_gradients([a[:32]], 1.0, out=[a[16:48]])
    with pytest.raises(ValueError, match="overlaps"):
        wide = torch.ones(4, 8, device=device)
        clip_gradients([wide[:, :3], wide[:, :3]], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_gradients([a], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_gradients([a], float("nan"))
    with pytest.raises(ValueError, match="shapes"):
        clip_gradients([a], 1.0, out=[b.half()])
    with pytest.raises(ValueError, match="one tensor"):
        clip_gradients([a], 1.0, out=[])
    with pytest.raises(TypeError):
        clip_gradients([a.double()], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_gradients([a.cpu()], 1.0)
    with pytest.raises(RuntimeError, match="require grad"):
        clip_gradients([torch.nn.Parameter(a)], 1.0)
    assert gradient_norm([]).item() == 0.0 and clip_gradients([], 1.0).item() == 0.0
    assert bool((a == 1).all()) and bool((b == 1).all())


def test_captured(device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    grads = [g.to(device) for g in _grads((5000, 3, 70_001), (BF16, F32))]
    outs = [torch.empty_like(g) for g in grads]
    clip_gradients(grads, 1.0, out=outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(grads, 1.0, out=outs)
    for seed in range(3):
        for g, new in zip(grads, _grads((5000, 3, 70_001), (BF16, F32), seed=seed, std=3.0 ** seed)):
            g.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [norm.clone(), *(o.clone() for o in outs)]
        eager = [torch.empty_like(g) for g in grads]
        want = [clip_gradients(grads, 1.0, out=eager), *eager]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_the_engine_clips_what_it_assigns(device):
    """``ScanADEngine(max_grad_norm=)`` leaves the clipped gradients on the parameters, the whole ones in the map."""
    from latent_bounded_interfaces_amd.backends import HipTransformerLowering
    from latent_bounded_interfaces_amd.backward import ScanADEngine, clip_grad_map
    from oracle import lbi_model as olbi

    model = olbi.OracleLBIModel(vocab_size=61, dim=32, n_heads=4, n_kv_heads=2, layers=4, layers_per_region=2, interface_width=8, hidden=48,
                                d_conv=4, interface_hidden=12, seed=31, lowering=HipTransformerLowering()).to(device)
    ids = torch.randint(0, 61, (2, 10), generator=torch.Generator().manual_seed(3)).to(device)
    whole = None
    for max_norm in (None, 0.01):
        logits, cache = model.forward_with_cache(ids)
        result = ScanADEngine(max_grad_norm=max_norm).backward(model=model, loss=olbi.token_loss(logits, ids), cache=cache)
        grads = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
        if max_norm is None:
            assert "grad_norm" not in result.diagnostics
            whole = grads
    assert set(grads) == set(whole)
    names = list(whole)
    want_norm, want = truth.clip([whole[n].cpu() for n in names], 0.01)
    assert float(want_norm[0]) > 0.01
    truth.assert_near(result.diagnostics["grad_norm"], want_norm)
    for n, one in zip(names, want):
        truth.assert_near(grads[n], one, n)
        assert torch.equal(result.grad_map[n], whole[n])
    clip_grad_map(result.grad_map, 0.01)
    for n in names:
        assert torch.equal(result.grad_map[n], grads[n])
