"""Calls of the clipping beside those of its own tests, against 64 bits with bounds by arithmetic (oracle/mlp_half.py)."""
from __future__ import annotations

import pytest
import torch

from oracle import mlp_half as truth

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _randn(seed, *shape, std=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std


def test_strided_results_that_share_memory_are_refused(device):
    """Results that lie on each other or on another gradient in part, or twice on themselves: nothing is written."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    grads, outs = _randn(1, 4, 8).to(device), torch.zeros(4, 8, device=device)
    alone, square = _randn(2, 7).to(device), _randn(3, 6, 6).to(device)
    calls = [
        ([grads[:, :3], grads[:, 3:6]], [outs[:, :3], outs[:, 2:5]]),
        ([grads[:, :4], grads[:, 4:]], [grads[:, 1:5], outs[:, 4:]]),
        ([grads[:, :4], grads[:, 4:]], [grads[:, 4:], grads[:, :4]]),
        ([grads[:, :4], alone], [grads[:, 1:5], torch.empty_like(alone)]),
        ([grads, alone], [outs[:, :1].expand(4, 8), torch.empty_like(alone)]),
        ([alone, grads[:, :3], grads[0, :3]], [torch.empty_like(alone), outs[:, :3], outs[0, :3]]),
        ([square, alone], [square.t(), torch.empty_like(alone)]),
    ]
    for got, into in calls:
        before = [t.clone() for t in (grads, outs, alone, square)]
        with pytest.raises((ValueError, RuntimeError), match="overlaps|share"):
            clip_gradients(got, 0.5, out=into)
        for a, b in zip((grads, outs, alone, square), before):
            assert torch.equal(a, b)
    spread = alone[:1].expand(5)
    before = alone.clone()
    with pytest.raises(ValueError, match="share"):
        clip_gradients([alone[2:], spread], 0.5)
    assert torch.equal(alone, before)


def test_parts_of_one_storage(device):
    """Results that lie between each other's elements, and some on their own gradients, are not refused."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    whole = _randn(4, 6, 12)
    base, twin = whole.to(device), torch.zeros(6, 12, device=device)
    cut = lambda t: [t[:, 0::3], t[:, 1::3], t[:2, 2::3], t[2:, 2::3]]
    want_norm, want = truth.clip(cut(whole), 1.0)
    truth.assert_near(clip_gradients(cut(base), 1.0, out=[*cut(base)[:2], *cut(twin)[2:]]), want_norm)
    for got, one in zip([*cut(base)[:2], *cut(twin)[2:]], want):
        truth.assert_near(got, one)
    for got, one in zip(cut(base)[2:], cut(whole)[2:]):
        assert torch.equal(got.cpu(), one)


@pytest.mark.parametrize("place", ["in place", "out", "strided"])
def test_a_backward_pass_that_saved_what_clipping_wrote_is_refused(place, device):
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients, gradient_norm

    leaf = torch.ones(6, 5, device=device, requires_grad=True)
    saved = _randn(5, 6, 5).to(device) if place != "strided" else _randn(5, 6, 9).to(device)[:, :5]
    product = (leaf * saved).sum()
    gradient_norm([saved])  # writes nothing
    product.backward(retain_graph=True)
    if place == "out":
        clip_gradients([_randn(6, 6, 5).to(device)], 0.5, out=[saved])
    else:
        clip_gradients([saved], 0.5)
    with pytest.raises(RuntimeError, match="inplace"):
        product.backward()


@pytest.mark.filterwarnings("ignore::DeprecationWarning")  # torch's own, where it first makes a tensor with a tangent
def test_derivatives_that_would_be_lost_are_refused(device):
    import torch.autograd.forward_ad as forward_ad

    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients, gradient_norm

    plain, other = _randn(7, 9).to(device), _randn(8, 3, 4).to(device)
    for grads in ([plain.clone().requires_grad_(), other], [plain, other.clone().requires_grad_()], [plain, other.t().clone().requires_grad_().t()]):
        outs = [torch.empty_like(g) for g in grads]
        with pytest.raises(RuntimeError, match="gradient_norm records no autograd graph"):
            gradient_norm(grads)
        with pytest.raises(RuntimeError, match="clip_gradients records no autograd graph"):
            clip_gradients(grads, 1.0, out=outs)
        with pytest.raises(RuntimeError, match="require grad"):
            clip_gradients(grads, 1.0)
        with torch.no_grad():
            assert torch.equal(gradient_norm(grads), clip_gradients(grads, 1.0, out=outs))
    with forward_ad.dual_level():
        dual = [plain, forward_ad.make_dual(other, torch.ones_like(other))]
        for call in (lambda: gradient_norm(dual), lambda: clip_gradients(dual, 1.0, out=[torch.empty_like(plain), torch.empty_like(other)]),
                     lambda: clip_gradients([plain], 1.0, out=[forward_ad.make_dual(plain.clone(), plain)]), lambda: clip_gradients(dual, 1.0)):
            with pytest.raises(RuntimeError, match="records no autograd graph"):
                call()
        gradient_norm([plain, other])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("max_norm,std", [(1.0, 3e37), (1e-3, 1e37), (1e-30, 1e9), (1e-38, 1e3), (0.0, 1.0), (2.0 ** -126, 0.25)])
def test_factors_below_the_smallest_normal_number(max_norm, std, dtype, device):
    """The factor's digits are not those that fp32 has left there."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    max_norm = float(torch.tensor(max_norm))  # as the call takes it
    for count in (4001, 16):
        grads = [_randn(9, count, std=std).to(dtype), _randn(10, 33, std=std)]
        assert all(bool(torch.isfinite(g).all()) for g in grads)
        _, want = truth.clip(grads, max_norm)
        outs = [torch.empty_like(g, device=device) for g in grads]
        clip_gradients([g.to(device) for g in grads], max_norm, out=outs)
        for got, one in zip(outs, want):
            truth.assert_near(got, one)


@pytest.mark.parametrize("max_norm", [2.0, 1e6])
def test_in_place_results_of_every_layout(max_norm, device):
    """Tensors off the vector grid, transposed, strided, of no and of one element, clipped where they are; what lies beside them is left as it was."""
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients

    flat, base, wide = _randn(11, 50_009).to(BF16), _randn(12, 64, 96), _randn(13, 40, 50).to(F16)
    parts = lambda f, b, w: [f[1:20_002], f[20_002:50_004], b[:, :60].t(), w[:, 3:20], f[50_004:50_004], f[50_006:50_007], w[5, 30:41]]
    on = [t.to(device) for t in (flat, base, wide)]
    want_norm, want = truth.clip(parts(flat, base, wide), max_norm)
    truth.assert_near(clip_gradients(parts(*on), max_norm), want_norm)
    for got, one in zip(parts(*on), want):
        truth.assert_near(got, one)
    for now, before in zip(on, (flat, base, wide)):
        kept = now.cpu()
        for part, old in zip(parts(kept, base, wide) if now is on[0] else parts(flat, kept, wide) if now is on[1] else parts(flat, base, kept),
                             parts(flat, base, wide)):
            part.copy_(old)
        assert torch.equal(kept, before)
