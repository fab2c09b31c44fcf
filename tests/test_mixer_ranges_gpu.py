"""Linear attention in half precision over the sizes that its inputs and states may have, on the GPU against the formulas in 64 bits.

fp32 results are held to bounds that shrink with the inputs: no tolerance here has an absolute part that they do not set."""
from __future__ import annotations

import pytest
import torch

import test_mixer_gpu as base
from latent_bounded_interfaces_amd.hip.transformer.mixer import linear_attention, linear_attention_input_pullback_basis
from oracle import mixer_half as oracle

pytestmark = pytest.mark.gpu

F16, F32 = base.F16, base.F32
STEP32 = base.STEP32


def summed(b, c):
    """What the lower ends of half precision can take from a sum of ``b_t c_t^T``: the decayed ``c`` of a column is scaled so that its largest is 2^13 at least,
    its second plane ends at 2^-24, half a step of which is 2^-38 of the largest."""
    return 2.0 ** -38 * b.abs().sum(-2)[..., :, None] * c.abs().amax(-2)[..., None, :]


@pytest.mark.parametrize("of_k, of_v", [(1.0, 1.0), (1.0, 1e-3), (1.0, 1e-5), (1e-3, 1e-5), (1e-5, 100.0)])
@pytest.mark.parametrize("shape", [(1, 2, 1, 130, 64, 64), (2, 2, 2, 65, 128, 128), (1, 1, 1, 700, 40, 33)])
def test_states_of_small_values(device, shape, of_k, of_v):
    gen = torch.Generator().manual_seed(40)
    q, k, v, log_decay, _ = base.inputs(gen, *shape, F16)
    k, v = (k.float() * of_k).to(F16), (v.float() * of_v).to(F16)
    out, final = linear_attention(*base.on(device, q, k, v, log_decay), scale=0.125)
    base.check_forward(q, k, v, log_decay, None, None, 0.125, out, None)
    group = q.shape[1] // k.shape[1]
    dq, dk, dv = base.d64(q, k, v)
    want = oracle.linear_attention(dq, dk, dv, log_decay, scale=1.0)[1]
    sizes = oracle.linear_attention(dq, dk.abs(), dv.abs(), log_decay, scale=1.0)[1]
    count = shape[3] + shape[5] + 16
    floor = summed(dk.repeat_interleave(group, 1), dv.repeat_interleave(group, 1))
    base.close(final, want, (2.0 ** -21 + count * STEP32) * sizes + floor, "state")


@pytest.mark.parametrize("of_q, of_g", [(1.0, 1.0), (1.0, 1e-3), (1.0, 1e-5), (1e-3, 1e-5), (1e-5, 100.0)])
@pytest.mark.parametrize("shape, basis", [((1, 2, 1, 130, 64, 64), 2), ((1, 1, 1, 700, 128, 96), 1)])
def test_cotangents_of_states_of_small_values(device, shape, basis, of_q, of_g):
    gen = torch.Generator().manual_seed(41)
    q, k, v, log_decay, first = base.inputs(gen, *shape, F16, state=True)
    bsz, heads, _, seqlen, _, dv = shape
    q = (q.float() * of_q).to(F16)
    g = base.rand(gen, bsz, basis, heads, seqlen, dv, dtype=F32, std=of_g).to(F16)
    scale = 0.125
    d_state = linear_attention_input_pullback_basis(*base.on(device, q, k, v, g, log_decay), scale=scale, state=first.to(device))[3]
    decay = log_decay.double().exp()[:, None] ** torch.arange(1, seqlen + 1)  # of out_t with respect to the first state
    count = seqlen + max(shape[4], dv) + 16
    for p in range(basis):
        a, b = q.double() * decay[..., None] * scale, g[:, p].double()
        want, sizes = a.mT @ b, a.abs().mT @ b.abs()
        base.close(d_state[:, p], want, (2.0 ** -20 + count * STEP32) * sizes + scale * summed(q.double(), b), "d_state")
