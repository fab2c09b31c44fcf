"""Linear attention and rotary positions on the GPU against their formulas in 64 bits.

Tolerances count roundings, each at most half a step u of the type: the result's own, and where an operator rounds operands in between, those, by
the magnitudes that they meet (oracle.mixer_half.rounded_operands).  What is fp32 throughout may be off by half an fp32 step for each addition."""
from __future__ import annotations

import math

import pytest
import torch

from latent_bounded_interfaces_amd.hip.transformer.mixer import (linear_attention, linear_attention_input_pullback_basis, linear_attention_step,
                                                                 rotary_heads, rotary_heads_pullback, rotary_tables)
from oracle import mixer_half as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(gen, *shape, dtype=BF16, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def close(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    if got.numel():
        over = (got - want).abs() - tol
        assert over.max() <= 0, (what, float(over.max()), float((got - want).norm() / want.norm().clamp(min=1e-300)))


def inputs(gen, bsz, heads, kv_heads, seqlen, dk, dv, dtype, *, state=False, memory=(1.0, 7.0), std=1.0):
    q, k, v = (rand(gen, bsz, h, seqlen, d, dtype=dtype, std=std) for h, d in ((heads, dk), (kv_heads, dk), (kv_heads, dv)))
    log_decay = -(2.0 ** -torch.linspace(*memory, heads))
    first = rand(gen, bsz, heads, dk, dv, dtype=F32) if state else None
    return q, k, v, log_decay, first


def on(device, *tensors):
    return tuple(None if t is None else t.to(device) for t in tensors)


def d64(*tensors):
    return tuple(None if t is None else t.double() for t in tensors)


def check_forward(q, k, v, log_decay, first, lengths, scale, out, state):
    dtype, u = q.dtype, half_step(q.dtype)
    dq, dk, dv, ds = d64(q, k, v, first)
    want, final = oracle.linear_attention(dq, dk, dv, log_decay, scale=scale, state=ds, lengths=lengths)
    group = q.shape[1] // k.shape[1]
    kk, vv = dk.repeat_interleave(group, 1), dv.repeat_interleave(group, 1)
    kk, vv = torch.nan_to_num(kk, 0, 0, 0), torch.nan_to_num(vv, 0, 0, 0)
    moved = oracle.rounded_operands(torch.nan_to_num(dq, 0, 0, 0), kk, vv, log_decay, first, lengths=lengths) * abs(scale)
    # the sums and weights in fp32, and the 16 (fp16: 22) bits of the decayed values, against magnitudes that no cancellation lowers
    count = q.shape[2] + q.shape[3] + 16
    rest = (2.0 ** -16 if dtype == BF16 else 2.0 ** -21) + count * STEP32
    sizes, of_state = oracle.linear_attention(torch.nan_to_num(dq, 0, 0, 0).abs(), kk.abs(), vv.abs(), log_decay, scale=abs(scale),
                                              state=None if ds is None else ds.abs(), lengths=lengths)
    smallest = 2.0 ** -24 if dtype == F16 else 0.0  # half precision's steps do not shrink below 2^-14
    close(out, want, u * (want.abs() + moved) * (1 + 4 * u) + rest * sizes + smallest * (1 + abs(scale) * q.shape[3]), "out")
    if state is not None:
        close(state, final, (2.0 ** -21 + count * STEP32) * of_state + (2.0 ** -24 * 8 if dtype == F16 else 1e-30), "state")


SHAPES = [  # B, H, Hkv, T, Dk, Dv
    (2, 2, 2, 1, 64, 64), (1, 3, 1, 2, 64, 128), (2, 4, 2, 63, 128, 64), (1, 2, 2, 64, 128, 128), (3, 2, 1, 65, 64, 64), (1, 2, 2, 127, 128, 128),
    (1, 4, 1, 130, 72, 40), (2, 1, 1, 200, 33, 7), (1, 2, 2, 129, 1, 1), (1, 1, 1, 97, 100, 128), (2, 2, 2, 449, 64, 64), (1, 2, 1, 600, 128, 128),
    (1, 1, 1, 300, 8, 120),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
def test_prompts(device, shape, dtype, state):
    gen = torch.Generator().manual_seed(hash((shape, state)) % 1000)
    q, k, v, log_decay, first = inputs(gen, *shape, dtype, state=state)
    scale = shape[4] ** -0.5
    out, final = linear_attention(*on(device, q, k, v, log_decay), scale=scale, state=on(device, first)[0])
    check_forward(q, k, v, log_decay, first, None, scale, out, final)
    again, nothing = linear_attention(*on(device, q, k, v, log_decay), scale=scale, state=on(device, first)[0], return_state=False)
    assert nothing is None
    check_forward(q, k, v, log_decay, first, None, scale, again, None)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("seqlen", [70, 400])
def test_lengths_and_what_lies_behind_them(device, dtype, wide, seqlen):
    gen = torch.Generator().manual_seed(5)
    lengths = torch.tensor([0, 1, 64, seqlen, seqlen - 3, 65], dtype=wide)
    q, k, v, log_decay, first = inputs(gen, 6, 2, 1, seqlen, 64, 80, dtype, state=True)
    for n in range(6):
        for t, bad in ((q, math.nan), (k, math.inf), (v, -math.inf)):
            t[n, :, int(lengths[n]):] = bad
    out, final = linear_attention(*on(device, q, k, v, log_decay), scale=0.3, state=first.to(device), lengths=lengths.to(device))
    check_forward(q, k, v, log_decay, first, lengths, 0.3, out, final)
    for n in range(6):
        assert (out[n, :, int(lengths[n]):] == 0).all()
    assert torch.equal(final[0].cpu(), first[0])
    # more than there are, and fewer than none
    odd = torch.tensor([-5, 1, 64, 1 << 30, seqlen - 3, 65], dtype=wide)
    for got, want in zip(linear_attention(*on(device, q, k, v, log_decay), scale=0.3, state=first.to(device), lengths=odd.to(device)), (out, final)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("decay", [0.0, -math.inf, -60.0, -1e-6])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decays_at_the_ends(device, decay, dtype):
    gen = torch.Generator().manual_seed(6)
    q, k, v, _, first = inputs(gen, 1, 2, 2, 330, 64, 64, dtype, state=True)
    log_decay = torch.full((2,), decay)
    out, final = linear_attention(*on(device, q, k, v, log_decay), scale=0.125, state=first.to(device))
    check_forward(q, k, v, log_decay.clamp(min=-1e4), first, None, 0.125, out, final)


def test_half_precision_past_its_largest_number(device):
    """Scores and states of millions, results of hundreds."""
    gen = torch.Generator().manual_seed(7)
    q, k, v, log_decay, _ = inputs(gen, 1, 2, 2, 200, 64, 64, F16, std=300.0)
    out, final = linear_attention(*on(device, q, k, v, log_decay), scale=1e-6)
    assert final.abs().max() > 65504
    check_forward(q, k, v, log_decay, None, None, 1e-6, out, final)


def test_half_precision_scores_of_nothing_beside_a_large_state(device):
    """Keys of zero in whole tiles, a state of 2^20 in front of them and queries of hundreds: neither's scale is the other's."""
    gen = torch.Generator().manual_seed(21)
    q, k, v, log_decay, first = inputs(gen, 1, 2, 2, 150, 64, 64, F16, state=True)
    k[:, :, :100] = 0
    q, first = q * 100, first * 2.0 ** 20
    out, final = linear_attention(*on(device, q, k, v, log_decay), scale=1e-7, state=first.to(device))
    check_forward(q, k, v, log_decay, first, None, 1e-7, out, final)


def test_offsets_past_32_bits(device):
    gen = torch.Generator().manual_seed(22)
    q, k, v, log_decay, _ = on(device, *inputs(gen, 1, 2, 2, 70, 64, 64, BF16))
    want = linear_attention(q, k, v, log_decay, scale=0.125) + linear_attention_input_pullback_basis(q, k, v, q[:, None], log_decay, scale=0.125)[:3]
    for strides in ((0, (1 << 31) + 64, 64, 1), (0, 64, (1 << 25) + 8, 1)):  # heads, then tokens, far apart
        far = torch.empty(1 + sum((n - 1) * s for n, s in zip((1, 2, 70, 64), strides)), dtype=BF16, device=device)
        views = [far.as_strided((1, 2, 70, 64), strides)]
        for i, t in enumerate((q, k, v)):
            views[0].copy_(t)
            args = [q, k, v]
            args[i] = views[0]
            got = linear_attention(*args, log_decay, scale=0.125) + linear_attention_input_pullback_basis(*args, q[:, None], log_decay, scale=0.125)[:3]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (strides, i)
        del far, views


def test_one_cotangent_for_all_tokens_and_many_directions(device):
    gen = torch.Generator().manual_seed(23)
    q, k, v, log_decay, _ = on(device, *inputs(gen, 2, 2, 1, 80, 64, 32, BF16))
    g = rand(gen, 2, 3, 2, 1, 32).to(device).expand(-1, -1, -1, 80, -1)
    for a, b in zip(linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=0.125)[:3],
                    linear_attention_input_pullback_basis(q, k, v, g.contiguous(), log_decay, scale=0.125)[:3]):
        assert torch.equal(a, b)
    # more chains than a launch numbers in its second dimension
    q, k, v, log_decay, _ = on(device, *inputs(gen, 1, 2, 2, 3, 8, 8, BF16))
    g = rand(gen, 1, 12000, 2, 3, 8).to(device)
    got = linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=0.5)
    some = linear_attention_input_pullback_basis(q, k, v, g[:, 11990:], log_decay, scale=0.5)
    assert all(torch.equal(a[:, 11990:], b) for a, b in zip(got[:3], some[:3]))


def test_strides(device):
    gen = torch.Generator().manual_seed(8)
    packed = rand(gen, 2, 150, (4 + 2 * 2) * 64).to(device)
    heads = packed.unflatten(-1, (-1, 64)).transpose(1, 2)
    q, k, v = heads[:, :4], heads[:, 4:6], heads[:, 6:]
    log_decay = torch.tensor([-0.5, -0.1, -0.02, -0.004], device=device)
    want = linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), log_decay, scale=0.125)
    for got in (linear_attention(q, k, v, log_decay, scale=0.125), linear_attention(q.flip(-1).flip(-1), k, v, log_decay, scale=0.125)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # rows that start on odd elements, a head dimension that is cut out, one key for all tokens
    wide = rand(gen, 2, 4, 150, 67).to(device)
    odd = wide[..., 1:65]
    same = linear_attention(odd, k, v, log_decay, scale=0.125)
    assert all(torch.equal(a, b) for a, b in zip(same, linear_attention(odd.contiguous(), k, v, log_decay, scale=0.125)))
    one = k[:, :, :1].expand(-1, -1, 150, -1)
    assert all(torch.equal(a, b) for a, b in zip(linear_attention(q, one, v, log_decay, scale=0.125),
                                                 linear_attention(q, one.contiguous(), v, log_decay, scale=0.125)))
    g = rand(gen, 2, 3, 150, 4, 64).to(device).transpose(2, 3)
    for a, b in zip(linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=0.125)[:3],
                    linear_attention_input_pullback_basis(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), log_decay, scale=0.125)[:3]):
        assert torch.equal(a, b) and a.is_contiguous()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 2, 2, 64, 64), (3, 4, 1, 128, 128), (2, 3, 3, 17, 33), (300, 4, 2, 64, 128), (1, 1, 1, 1, 1), (200, 2, 2, 100, 60)])
def test_tokens(device, shape, dtype):
    bsz, heads, kv_heads, dk, dv = shape
    gen = torch.Generator().manual_seed(9)
    q, k, v = rand(gen, bsz, heads, dk, dtype=dtype), rand(gen, bsz, kv_heads, dk, dtype=dtype), rand(gen, bsz, kv_heads, dv, dtype=dtype)
    log_decay, state = -torch.rand(heads, generator=gen), rand(gen, bsz, heads, dk, dv, dtype=F32)
    active = torch.rand(bsz, generator=gen) < 0.7
    mine, version = state.to(device), None
    version = mine._version
    out = linear_attention_step(*on(device, q, k, v, log_decay), mine, scale=0.5, active=active.to(device))
    assert mine._version > version
    want, after = oracle.linear_attention(*(t.double()[:, :, None] for t in (q, k, v)), log_decay, scale=0.5, state=state.double())
    want = torch.where(active[:, None, None], want[:, :, 0], 0.0)
    after = torch.where(active[:, None, None, None], after, state.double())
    sizes = oracle.linear_attention(*(t.double().abs()[:, :, None] for t in (q, k, v)), log_decay, scale=0.5, state=state.double().abs())
    close(out, want, half_step(dtype) * want.abs() + (dk + 8) * STEP32 * sizes[0][:, :, 0] + (2.0 ** -25 if dtype == F16 else 0.0), "out")
    close(mine, after, 8 * STEP32 * sizes[1], "state")
    assert torch.equal(mine.cpu()[~active], state[~active]) and (out.cpu()[~active] == 0).all()


def test_a_prompt_in_pieces_and_then_token_by_token(device):
    gen = torch.Generator().manual_seed(10)
    q, k, v, log_decay, _ = inputs(gen, 2, 4, 2, 170, 64, 64, BF16)
    dq, dk, dv, dl = on(device, q, k, v, log_decay)
    state, rows = None, []
    for piece in (slice(0, 70), slice(70, 71), slice(71, 160)):
        # Each piece's 64 tokens are counted from its own first one, so its roundings are those of a call of its own: the pair of tokens 64 and 71, say, is a
        # rounded score in the whole and reaches token 71 through the rounded copy of the state here.
        before = state
        out, state = linear_attention(dq[:, :, piece], dk[:, :, piece], dv[:, :, piece], dl, scale=0.125, state=before)
        check_forward(q[:, :, piece], k[:, :, piece], v[:, :, piece], log_decay, None if before is None else before.cpu(), None, 0.125, out, state)
        rows.append(out)
    for t in range(160, 170):
        rows.append(linear_attention_step(dq[:, :, t], dk[:, :, t], dv[:, :, t], dl, state, scale=0.125)[:, :, None])
    want, final = oracle.linear_attention(*d64(q, k, v), log_decay, scale=0.125)
    _, of_state = oracle.linear_attention(*(t.double().abs() for t in (q, k, v)), log_decay, scale=0.125)
    close(state, final, (2.0 ** -21 + (170 + 64) * STEP32) * of_state, "state")
    # three roundings of half a step at most: the scores, the state's copy, the result
    assert (torch.cat(rows, 2).cpu().double() - want).norm() <= 3 * half_step(BF16) * want.norm()


def check_pullback(q, k, v, g, log_decay, scale, first, g_state, lengths, got):
    dtype, u = q.dtype, half_step(q.dtype)
    bsz, heads, seqlen, dk = q.shape
    group, count = heads // k.shape[1], seqlen + max(dk, v.shape[-1]) + 16
    qq, kk, vv, gg = (torch.nan_to_num(t.double(), 0, 0, 0) for t in (q, k, v, g))
    kk, vv = kk.repeat_interleave(group, 1), vv.repeat_interleave(group, 1)
    rest = (2.0 ** -16 if dtype == BF16 else 2.0 ** -21) + count * STEP32
    for p in range(g.shape[1]):
        leaves = [t.clone().requires_grad_() for t in (qq, kk, vv)] + ([first.double().requires_grad_()] if first is not None else [])
        out, final = oracle.linear_attention(*leaves[:3], log_decay, scale=scale, state=leaves[3] if first is not None else None, lengths=lengths)
        gp = gg[:, p]
        total = (out * gp).sum() + (0.0 if g_state is None else (final * g_state[:, p].double()).sum())
        want = torch.autograd.grad(total, leaves)
        gs = None if g_state is None else g_state[:, p].double() / scale
        moved = [oracle.rounded_operands(gp, vv, kk, log_decay, None if first is None else first.mT, lengths=lengths),
                 oracle.rounded_operands(vv, gp, qq, log_decay, None if gs is None else gs.mT, lengths=lengths, reverse=True, shift=1),
                 oracle.rounded_operands(kk, qq, gp, log_decay, gs, lengths=lengths, reverse=True, shift=1)]
        # magnitudes: the same gradients of magnitudes
        leaves = [t.abs().requires_grad_() for t in (qq, kk, vv)] + ([first.double().abs().requires_grad_()] if first is not None else [])
        out, final = oracle.linear_attention(*leaves[:3], log_decay, scale=abs(scale), state=leaves[3] if first is not None else None, lengths=lengths)
        sizes = torch.autograd.grad((out * gp.abs()).sum() + (0.0 if g_state is None else (final * g_state[:, p].double().abs()).sum()), leaves)
        smallest = 2.0 ** -24 * (1 + abs(scale) * 128) if dtype == F16 else 0.0
        for i, name in enumerate(("dq", "dk", "dv")):
            close(got[i][:, p], want[i], u * (want[i].abs() + abs(scale) * moved[i]) * (1 + 4 * u) + rest * sizes[i] + smallest, name)
        if first is not None:
            close(got[3][:, p], want[3], (2.0 ** -20 + count * STEP32) * sizes[3] + (2.0 ** -21 if dtype == F16 else 1e-30), "d_state")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape, basis", [((1, 2, 2, 64, 64, 64), 1), ((2, 2, 1, 65, 64, 64), 3), ((1, 2, 2, 130, 128, 128), 2), ((1, 2, 2, 90, 128, 64), 2),
                                          ((1, 1, 1, 70, 40, 72), 1), ((2, 3, 1, 5, 7, 33), 2), ((1, 2, 2, 500, 64, 64), 1), ((1, 1, 1, 1, 64, 64), 4)])
@pytest.mark.parametrize("state", [False, True])
def test_pullback(device, shape, basis, dtype, state):
    gen = torch.Generator().manual_seed(11)
    q, k, v, log_decay, first = inputs(gen, *shape, dtype, state=state)
    bsz, heads, _, seqlen, dk, dv = shape
    g = rand(gen, bsz, basis, heads, seqlen, dv, dtype=dtype)
    g_state = rand(gen, bsz, basis, heads, dk, dv, dtype=F32) if state else None
    scale = dk ** -0.5
    got = linear_attention_input_pullback_basis(*on(device, q, k, v, g, log_decay), scale=scale, state=on(device, first)[0],
                                                g_state=on(device, g_state)[0])
    assert (got[3] is None) == (first is None)
    check_pullback(q, k, v, g, log_decay, scale, first, g_state, None, got)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_pullback_with_lengths(device, dtype):
    gen = torch.Generator().manual_seed(12)
    lengths = torch.tensor([0, 1, 64, 140, 75])
    q, k, v, log_decay, first = inputs(gen, 5, 2, 2, 140, 64, 48, dtype, state=True)
    g, g_state = rand(gen, 5, 2, 2, 140, 48, dtype=dtype), rand(gen, 5, 2, 2, 64, 48, dtype=F32)
    for n in range(5):
        for t in (q, k, v):
            t[n, :, int(lengths[n]):] = math.nan
        g[n, :, :, int(lengths[n]):] = math.inf
    got = linear_attention_input_pullback_basis(*on(device, q, k, v, g, log_decay), scale=0.2, state=first.to(device), g_state=g_state.to(device),
                                                lengths=lengths.to(device))
    check_pullback(q, k, v, g, log_decay, 0.2, first, g_state, lengths, got)
    for n in range(5):
        for t in got[:3]:
            assert (t[n, :, :, int(lengths[n]):] == 0).all()


# chains that are cut in two, whose states come in halves; in three; and in so many that a launch joins their states
@pytest.mark.parametrize("bsz, heads, seqlen", [(4, 24, 2100), (5, 16, 1500), (5, 1, 2500)])
def test_long_sequences_of_some_length_in_many_chains(device, bsz, heads, seqlen):
    gen = torch.Generator().manual_seed(29)
    lengths = torch.tensor([0, 1100, seqlen, 40, 700][:bsz])
    q, k, v, log_decay, first = inputs(gen, bsz, heads, heads, seqlen, 32, 24, BF16, state=True)
    for n in range(bsz):
        k[n, :, int(lengths[n]):] = math.nan
    out, final = linear_attention(*on(device, q, k, v, log_decay), scale=0.3, state=first.to(device), lengths=lengths.to(device))
    check_forward(q, k, v, log_decay, first, lengths, 0.3, out, final)
    for n in range(bsz):
        assert (out[n, :, int(lengths[n]):] == 0).all()


@pytest.mark.parametrize("bsz, heads, seqlen", [(4, 8, 2100), (3, 1, 2500)])
def test_pullback_of_long_sequences_of_some_length(device, bsz, heads, seqlen):
    gen = torch.Generator().manual_seed(30)
    lengths = torch.tensor([0, 1100, seqlen, 40][4 - bsz:])
    q, k, v, log_decay, first = inputs(gen, bsz, heads, heads, seqlen, 16, 16, BF16, state=True)
    g, g_state = rand(gen, bsz, 1, heads, seqlen, 16, dtype=BF16), rand(gen, bsz, 1, heads, 16, 16, dtype=F32)
    for n in range(bsz):
        q[n, :, int(lengths[n]):] = math.nan
        g[n, :, :, int(lengths[n]):] = math.inf
    got = linear_attention_input_pullback_basis(*on(device, q, k, v, g, log_decay), scale=0.2, state=first.to(device), g_state=g_state.to(device),
                                                lengths=lengths.to(device))
    check_pullback(q, k, v, g, log_decay, 0.2, first, g_state, lengths, got)


@pytest.mark.parametrize("seqlen", [0, 3])
@pytest.mark.parametrize("bsz", [0, 2])
def test_nothing_to_do(device, bsz, seqlen):
    gen = torch.Generator().manual_seed(13)
    q, k, v, log_decay, first = on(device, *inputs(gen, bsz, 2, 1, seqlen, 64, 32, BF16, state=True))
    out, final = linear_attention(q, k, v, log_decay, scale=1.0, state=first)
    assert out.shape == (bsz, 2, seqlen, 32) and final.shape == first.shape
    if not seqlen:
        assert torch.equal(final, first)
        assert linear_attention(q, k, v, log_decay, scale=1.0)[1].abs().sum() == 0
    for basis in (0, 2):
        grads = linear_attention_input_pullback_basis(q, k, v, q.new_zeros(bsz, basis, 2, seqlen, 32), log_decay, scale=1.0, state=first)
        assert [tuple(t.shape) for t in grads] == [(bsz, basis, 2, seqlen, 64)] * 2 + [(bsz, basis, 2, seqlen, 32), (bsz, basis, 2, 64, 32)]
        assert all((t == 0).all() for t in grads)


ROTARY = [  # B, T, H, Hkv, Dh, R
    (2, 5, 4, 2, 64, 64), (1, 1, 1, 1, 128, 128), (2, 33, 3, 1, 128, 64), (1, 7, 2, 2, 30, 10), (2, 3, 2, 1, 7, 6), (1, 4, 2, 2, 16, 0), (3, 6, 12, 12, 64, 48),
    (1, 9, 6, 3, 256, 16), (1, 5, 2, 1, 2, 2),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary(device, shape, interleaved, dtype):
    bsz, seqlen, heads, kv_heads, dim, rotary = shape
    gen = torch.Generator().manual_seed(14)
    cos, sin = rotary_tables(500, rotary, device="cpu")
    qkv = rand(gen, bsz, seqlen, (heads + 2 * kv_heads) * dim, dtype=dtype)
    u = half_step(dtype)
    for positions in (None, torch.randint(0, 500, (bsz, seqlen), generator=gen), torch.randint(0, 500, (seqlen,), generator=gen, dtype=torch.int32)):
        kinds = dict(n_heads=heads, n_kv_heads=kv_heads, interleaved=interleaved)
        got = rotary_heads(*on(device, qkv, cos, sin), **kinds, positions=on(device, positions)[0])
        want = oracle.rotary_heads(qkv.double(), cos.double(), sin.double(), **kinds, positions=positions)
        # two products and an addition in fp32, and one rounding; |x1| + |x2| is at most twice the largest
        slack = 3 * STEP32 * 2 * qkv.double().abs().max()
        for a, b in zip(got, want):
            close(a, b, u * b.abs() + slack + (2.0 ** -25 if dtype == F16 else 0.0))
        assert torch.equal(got[2].cpu(), want[2].to(dtype)) and got[0].is_contiguous() and got[1].is_contiguous()
        assert got[2].data_ptr() >= 0 and got[2].untyped_storage().nbytes() == qkv.untyped_storage().nbytes()
        for shared in {heads, kv_heads}:
            dq, dk, dv = (rand(gen, bsz, 2, h, seqlen, dim, dtype=dtype) for h in (heads, shared, shared))
            back = rotary_heads_pullback(*on(device, dq, dk, dv, cos, sin), n_kv_heads=kv_heads, interleaved=interleaved, positions=on(device, positions)[0])
            for p in range(2):
                leaf = qkv.double().requires_grad_()
                sums = [t[:, p].double() for t in (dq, dk, dv)]
                sums[1:] = [t.unflatten(1, (kv_heads, -1)).sum(2) for t in sums[1:]]
                outs = oracle.rotary_heads(leaf, cos.double(), sin.double(), **kinds, positions=positions)
                want_back, = torch.autograd.grad(sum((o * s).sum() for o, s in zip(outs, sums)), leaf)
                slack = (heads // kv_heads + 3) * STEP32 * 2 * (heads // kv_heads) * max(t.double().abs().max() for t in (dq, dk, dv))
                close(back[:, p], want_back, u * want_back.abs() + slack + (2.0 ** -25 if dtype == F16 else 0.0))


def test_rotary_positions_outside_the_tables(device):
    gen = torch.Generator().manual_seed(15)
    qkv = rand(gen, 1, 4, 3 * 32, dtype=F32).to(device)
    cos, sin = rotary_tables(10, 16, device=device)
    positions = torch.tensor([3, 10, -1, 9], device=device)
    q, k, v = rotary_heads(qkv, cos, sin, n_heads=1, n_kv_heads=1, positions=positions)
    for t in (q, k):
        assert torch.isnan(t[0, 0, 1:3, :16]).all() and torch.isfinite(t[0, 0, 1:3, 16:]).all() and torch.isfinite(t[0, 0, [0, 3]]).all()
    assert torch.isfinite(v).all()
    back = rotary_heads_pullback(q[:, None].nan_to_num(), k[:, None].nan_to_num(), v[:, None].contiguous(), cos, sin, n_kv_heads=1, positions=positions)
    assert torch.isnan(back[0, 0, 1:3, :16]).all() and torch.isfinite(back[0, 0, :, 64:]).all() and torch.isfinite(back[0, 0, [0, 3]]).all()


def test_rotary_of_strided_projections(device):
    gen = torch.Generator().manual_seed(16)
    cos, sin = rotary_tables(50, 64, device=device)
    wide = rand(gen, 20, 3, 4 * 64 + 8).to(device)
    for view in (wide[..., :256], wide[..., 3:259], wide[::2, :, :256], wide.transpose(0, 1)[..., :256]):
        got = rotary_heads(view, cos, sin, n_heads=2, n_kv_heads=1)
        for a, b in zip(got, rotary_heads(view.contiguous(), cos, sin, n_heads=2, n_kv_heads=1)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("shift", (1, 2, 5))
def test_tensors_that_start_on_any_element(device, shift, dtype):
    gen = torch.Generator().manual_seed(23)

    def shifted(t):
        room = torch.empty(t.numel() + shift, dtype=t.dtype, device=device)
        room[shift:].copy_(t.flatten())
        return room[shift:].view(t.shape)

    cos, sin = rotary_tables(70, 64, device=device)
    qkv, dq = rand(gen, 2, 70, 4 * 64, dtype=dtype).to(device), rand(gen, 2, 3, 2, 70, 64, dtype=dtype).to(device)
    for interleaved in (False, True):
        for a, b in zip(rotary_heads(shifted(qkv), cos, sin, n_heads=2, n_kv_heads=1, interleaved=interleaved),
                        rotary_heads(qkv, cos, sin, n_heads=2, n_kv_heads=1, interleaved=interleaved)):
            assert torch.equal(a, b)
        assert torch.equal(rotary_heads_pullback(shifted(dq), dq, shifted(dq), cos, sin, n_kv_heads=1, interleaved=interleaved),
                           rotary_heads_pullback(dq, dq, dq, cos, sin, n_kv_heads=1, interleaved=interleaved))
    if dtype == torch.float32:
        return
    q, g = dq[:, 0], dq
    log_decay = torch.tensor([-0.5, -0.01], device=device)
    for a, b in zip(linear_attention(shifted(q), q, shifted(q), log_decay, scale=0.125), linear_attention(q, q, q, log_decay, scale=0.125)):
        assert torch.equal(a, b)
    for a, b in zip(linear_attention_input_pullback_basis(shifted(q), q, q, shifted(g), log_decay, scale=0.125)[:3],
                    linear_attention_input_pullback_basis(q, q, q, g, log_decay, scale=0.125)[:3]):
        assert torch.equal(a, b)


def _layer(gen, bsz, seqlen, heads, kv_heads, dim, dtype):
    qkv = rand(gen, bsz, seqlen, (heads + 2 * kv_heads) * dim, dtype=dtype)
    cos, sin = rotary_tables(2048, dim // 2, base=500.0, device="cpu", factor=4.0, original_length=512)
    return qkv, cos, sin, -(2.0 ** -torch.linspace(1, 6, heads))


def test_from_the_projection_to_its_cotangent(device):
    """Rotary positions, linear attention and both pullbacks one after the other, as a layer runs them, against derivatives of all of it."""
    gen = torch.Generator().manual_seed(17)
    bsz, seqlen, heads, kv_heads, dim = 2, 100, 4, 2, 64
    qkv, cos, sin, log_decay = _layer(gen, bsz, seqlen, heads, kv_heads, dim, BF16)
    basis = rand(gen, bsz, 2, seqlen, heads * dim)
    x, c, s, l, g = on(device, qkv, cos, sin, log_decay, basis)
    q, k, v = rotary_heads(x, c, s, n_heads=heads, n_kv_heads=kv_heads)
    out, _ = linear_attention(q, k, v, l, scale=dim ** -0.5)
    merged = out.transpose(1, 2).flatten(2)
    assert merged.data_ptr() == out.data_ptr()  # no copy on the way to the output projection
    grads = linear_attention_input_pullback_basis(q, k, v, g.unflatten(-1, (heads, dim)).transpose(2, 3), l, scale=dim ** -0.5)
    back = rotary_heads_pullback(*grads[:3], c, s, n_kv_heads=kv_heads)
    leaf = qkv.double().requires_grad_()
    want_out = oracle.linear_attention(*oracle.rotary_heads(leaf, cos.double(), sin.double(), n_heads=heads, n_kv_heads=kv_heads), log_decay,
                                       scale=dim ** -0.5)[0].transpose(1, 2).flatten(2)
    # roundings of relative size 2^-8 at most: q, k, their decayed scores, the state's copy and the result; backwards q, k, the scores, the copy, three
    # results and the sum of the heads
    u = half_step(BF16)
    assert (merged.cpu().double() - want_out).norm() <= 5 * u * want_out.norm()
    for p in range(2):
        want, = torch.autograd.grad((want_out * basis[:, p].double()).sum(), leaf, retain_graph=True)
        assert (back[:, p].cpu().double() - want).norm() <= 6 * u * want.norm()


@pytest.mark.parametrize("bsz, seqlen", [(1, 700), (8, 130)])
def test_captured_and_replayed(device, bsz, seqlen):
    gen = torch.Generator().manual_seed(18)
    heads, kv_heads, dim = 4, 2, 64
    qkv, cos, sin, log_decay = on(device, *_layer(gen, bsz, seqlen, heads, kv_heads, dim, BF16))
    basis, first = rand(gen, bsz, 1, heads, seqlen, dim).to(device), rand(gen, bsz, heads, dim, dim, dtype=F32).to(device)
    lengths = torch.randint(0, seqlen + 1, (bsz,), generator=gen).to(device)

    def run(x, g, state, lengths):
        q, k, v = rotary_heads(x, cos, sin, n_heads=heads, n_kv_heads=kv_heads)
        out, after = linear_attention(q, k, v, log_decay, scale=0.125, state=state, lengths=lengths)
        grads = linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=0.125, state=state, lengths=lengths)
        back = rotary_heads_pullback(*grads[:3], cos, sin, n_kv_heads=kv_heads)
        token = linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], log_decay, after, scale=0.125)
        return out, after, back, grads[3], token

    x, g, s, n = qkv.clone(), basis.clone(), first.clone(), lengths.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, g, s, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = run(x, g, s, n)
    for turn in range(4):
        x.copy_(qkv * (1 + turn)), g.copy_(basis.roll(turn, 0) * (2 - turn)), s.copy_(first * turn), n.copy_(lengths.flip(0) if turn % 2 else lengths)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(results, run(x, g, s, n)):
            assert torch.equal(got, want), turn


def test_two_streams_at_once_and_reruns(device):
    gen = torch.Generator().manual_seed(19)
    q, k, v, log_decay, first = on(device, *inputs(gen, 1, 2, 2, 1500, 128, 128, BF16, state=True))
    g = rand(gen, 1, 2, 2, 1500, 128).to(device)
    torch.cuda.synchronize()
    want = linear_attention(q, k, v, log_decay, scale=0.1, state=first) + linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=0.1)[:3]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        results = []
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append(linear_attention(q, k, v, log_decay, scale=0.1, state=first)
                               + linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=0.1)[:3])
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_derivatives_are_refused(device):
    gen = torch.Generator().manual_seed(20)
    q, k, v, log_decay, first = on(device, *inputs(gen, 1, 2, 1, 5, 64, 64, BF16, state=True))
    g, qkv = q[:, None].clone(), rand(gen, 1, 5, 3 * 64).to(device)
    cos, sin = rotary_tables(5, 64, device=device)
    calls = {
        "linear_attention": lambda: linear_attention(q, k, v, log_decay, scale=1.0, state=first),
        "linear_attention_step": lambda: linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], log_decay, first, scale=1.0),
        "pullback": lambda: linear_attention_input_pullback_basis(q, k, v, g, log_decay, scale=1.0),
        "rotary_heads": lambda: rotary_heads(qkv, cos, sin, n_heads=1, n_kv_heads=1),
    }
    for leaf, names in ((log_decay, ("linear_attention", "linear_attention_step", "pullback")), (qkv, ("rotary_heads",))):
        leaf.requires_grad_()
        for name in names:
            with pytest.raises(RuntimeError, match="no_grad"):
                calls[name]()
            with torch.no_grad():
                calls[name]()
        leaf.requires_grad_(False)
