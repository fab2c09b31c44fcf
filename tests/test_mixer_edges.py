"""What linear attention's entry points refuse at the ends of their ranges, without a device."""
from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from latent_bounded_interfaces_amd import _lib
from latent_bounded_interfaces_amd.hip.transformer import block, mixer

OK = ctypes.c_void_p(256)  # never dereferenced


def call(**changed):
    sizes = dict(B=2, P=1, H=4, Hkv=2, T=100, Dk=64, Dv=64, q=256, k=256, v=256, q_stride=(25600, 6400, 64), k_stride=(12800, 6400, 64),
                 v_stride=(12800, 6400, 64), log_decay=256, out=256, out_stride=(25600, 64, 256), state_out=256, g_out=256,
                 g_out_stride=(25600, 25600, 6400, 64), dq=256, dk=256, dv=256, scale=1.0, dtype=_lib.LBI_BF16)
    return _lib.LinearAttentionCall(**{**sizes, **changed})


@pytest.mark.parametrize("scale", [2.0 ** -128, -(2.0 ** -149), 1e-50, 0.0, math.inf, 1e39, math.nan])
def test_a_scale_without_an_inverse(scale):
    lib = _lib.load()
    for entry in ("lbi_linear_attention", "lbi_linear_attention_pullback"):
        # (of no sequences: what is not refused has nothing to do)
        assert getattr(lib, entry)(ctypes.byref(call(B=0, scale=scale)), OK, 1 << 40, None) == -1 and b"scale" in lib.lbi_last_error(), entry
    h = torch.bfloat16
    q, k, v, log_decay = torch.zeros(2, 4, 5, 8, dtype=h), torch.zeros(2, 2, 5, 8, dtype=h), torch.zeros(2, 2, 5, 6, dtype=h), torch.zeros(4)
    with pytest.raises(ValueError, match="scale"):
        mixer.linear_attention(q, k, v, log_decay, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        mixer.linear_attention_input_pullback_basis(q, k, v, torch.zeros(2, 1, 4, 5, 6, dtype=h), log_decay, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        mixer.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], log_decay, torch.zeros(2, 4, 8, 6), scale=scale)


@pytest.mark.parametrize("scale", [2.0 ** -127, 2.0 ** -128 + 2.0 ** -149, -1e-38, 3e38])
def test_a_scale_with_one(scale):
    lib = _lib.load()
    for entry in ("lbi_linear_attention", "lbi_linear_attention_pullback"):
        assert getattr(lib, entry)(ctypes.byref(call(B=0, scale=scale)), OK, 1 << 40, None) == 0, entry
    token = torch.zeros(2, 4, 8), torch.zeros(2, 4, 8), torch.zeros(2, 4, 6)
    with pytest.raises(RuntimeError, match="CUDA"):
        mixer.linear_attention_step(*token, torch.zeros(4), torch.zeros(2, 4, 8, 6), scale=scale)


def test_more_chains_than_a_launch_has_workgroups_for():
    lib = _lib.load()
    least = 2 ** 24 - 8  # of 256 threads each, rounded up to eights: fewer than 2^32 threads

    def status(entry, **sizes):
        # (without log_decay: a call of sizes that are taken goes no further than that)
        got = getattr(lib, entry)(ctypes.byref(call(**{**dict(T=1, Dk=8, Dv=8, log_decay=None), **sizes})), OK, 1 << 40, None)
        return got, lib.lbi_last_error()

    for entry, sizes in (("lbi_linear_attention", dict(B=1 << 19, H=64, Hkv=64)), ("lbi_linear_attention", dict(B=1 << 19, H=32, Hkv=1)),
                         ("lbi_linear_attention_pullback", dict(B=1 << 10, H=16, P=1 << 9)), ("lbi_linear_attention_pullback", dict(B=1 << 10, H=16, P=512, Dv=4))):
        got, why = status(entry, **sizes)
        assert got == -2 and b"too many" in why, (entry, sizes)
        assert getattr(lib, entry + "_workspace_bytes")(ctypes.byref(call(**{**dict(T=1, Dk=8, Dv=8), **sizes}))) == 0
    for entry, sizes, chains in (("lbi_linear_attention", dict(B=6223, H=2696, Hkv=1), 1), ("lbi_linear_attention_pullback", dict(B=1 << 10, H=16, P=341), 3),
                                 ("lbi_linear_attention_pullback", dict(B=1 << 10, H=16, P=511, Dv=4), 2)):
        count = chains * sizes["B"] * sizes["H"] * sizes.get("P", 1)
        assert 0.99 * least < count <= least
        got, why = status(entry, **sizes)
        assert got == -1 and b"null" in why, (entry, sizes)


def test_how_many_rows_a_gate_has():
    """The type of a gate's gradient goes by what the gate is of, not by the number of positions."""
    d = 16
    for positions in ((1,), (5,), (1, 1), (2, 3)):
        branch = torch.zeros(3, *positions, d)
        of_sequence = torch.zeros(3, *[1] * len(positions), d)
        assert block._rows_of_gate("x", of_sequence, branch, True) == math.prod(positions)
        assert block._rows_of_gate("x", branch, branch) == 0
        for gate in (torch.zeros(d), torch.zeros(1, *[1] * len(positions), d), torch.zeros(3, *positions, 1), torch.zeros(3, d)):
            with pytest.raises(ValueError, match="gate must be"):
                block._rows_of_gate("x", gate, branch, True)
    with pytest.raises(ValueError, match="gate must be"):
        block._rows_of_gate("x", torch.zeros(3, d), torch.zeros(3, d), True)
    assert block._rows_of_gate("x", None, branch, True) == 0
    x, w = torch.zeros(2, 3, d), torch.ones(d)
    with pytest.raises(ValueError, match="gate must be"):
        block.gated_residual_rmsnorm_pullback(x, x, x, w, w, 1e-5, gate=x, sequence_gate=True)


def test_a_packed_call_is_the_structure():
    """The wrappers pack the call's bytes; the header's structure is what the entry points read."""
    names = [(name, getattr(kind, "_length_", 1)) for name, kind in _lib.LinearAttentionCall._fields_]
    whole = [n for n, count in names[:-3] for _ in range(count)]  # 8 bytes each
    assert [n for n, _ in names[-3:]] == ["scale", "dtype", "lengths_wide"] and len(whole) == 37
    packed = _lib.pack_linear_attention_call(*range(1000, 1037), 0.75, 2, 1)
    assert len(packed) == ctypes.sizeof(_lib.LinearAttentionCall)
    read = _lib.LinearAttentionCall.from_buffer_copy(packed)
    values = [v for name, count in names[:-3] for v in (list(getattr(read, name)) if count > 1 else [getattr(read, name)])]
    assert values == list(range(1000, 1037)) and (read.scale, read.dtype, read.lengths_wide) == (0.75, 2, 1)
    # and in the order in which the wrappers give them
    q, k, v = (torch.zeros(2, heads, 5, width, dtype=torch.bfloat16) for heads, width in ((4, 8), (2, 8), (2, 6)))
    log_decay, state, g_state, d_state = torch.zeros(4), torch.zeros(2, 4, 8, 6), torch.zeros(2, 3, 4, 8, 6), torch.zeros(2, 3, 4, 8, 6)
    lengths, out, state_out = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 5, 4, 6).transpose(1, 2), torch.zeros(2, 4, 8, 6)
    g, grads = torch.zeros(2, 3, 4, 5, 6), tuple(torch.zeros(2, 3, 4, 5, width) for width in (8, 8, 6))
    read = _lib.LinearAttentionCall.from_buffer_copy(mixer._call(q, k, v, log_decay, 0.5, state, lengths, basis=3, out=out, state_out=state_out, g_out=g,
                                                                 g_state=g_state, grads=grads, d_state=d_state))
    assert [getattr(read, n) for n in ("B", "P", "H", "Hkv", "T", "Dk", "Dv")] == [2, 3, 4, 2, 5, 8, 6]
    for name, t in dict(q=q, k=k, v=v, log_decay=log_decay, state=state, lengths=lengths, out=out, state_out=state_out, g_out=g, g_state=g_state, dq=grads[0],
                        dk=grads[1], dv=grads[2], d_state=d_state).items():
        assert getattr(read, name) == t.data_ptr(), name
    for name, t in dict(q_stride=q, k_stride=k, v_stride=v, out_stride=out, g_out_stride=g).items():
        assert list(getattr(read, name)) == list(t.stride()[:-1]), name
    assert (read.scale, read.dtype, read.lengths_wide) == (0.5, _lib.LBI_BF16, 1)
    # the header's own order
    header = (Path(__file__).resolve().parents[1] / "include" / "lbi_hip.h").read_text()
    body = re.search(r"typedef struct lbi_linear_attention_call \{(.*?)\}", header, re.S)[1]
    declared = [(m[1], int(m[2] or 1)) for part in body.split(";") for m in re.finditer(r"(\w+)(?:\[(\d)\])?\s*(?:,|$)", part.strip())]
    assert declared == names
