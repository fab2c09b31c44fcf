"""What the entry points of a linear-attention block's mixer half refuse, each with its status and before anything is launched; what their
Python wrappers refuse without a device; and the rotary tables."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from latent_bounded_interfaces_amd import _lib
from latent_bounded_interfaces_amd.hip.transformer import block, mixer

OK, ODD = ctypes.c_void_p(256), ctypes.c_void_p(257)  # never dereferenced
F32, F16, BF16 = _lib.LBI_F32, _lib.LBI_F16, _lib.LBI_BF16


def test_rotary_statuses():
    lib = _lib.load()

    def forward(qkv=OK, cos=OK, sin=OK, positions=None, q=OK, k=OK, B=2, T=3, H=4, Hkv=2, D=8, R=4, table=3, sb=384, st=64, wide=0, il=0, dtype=BF16):
        return lib.lbi_rotary(qkv, cos, sin, positions, q, k, B, T, H, Hkv, D, R, table, sb, st, wide, il, dtype, None), lib.lbi_last_error()

    def back(q=OK, k=OK, v=OK, cos=OK, sin=OK, positions=None, g=OK, B=2, P=1, T=3, H=4, Hkv=2, kv=4, D=8, R=4, table=3, wide=0, il=0, dtype=BF16):
        return (lib.lbi_rotary_pullback(q, k, v, cos, sin, positions, g, B, P, T, H, Hkv, kv, D, R, table, wide, il, dtype, None), lib.lbi_last_error())

    for call in (forward, back):
        assert call(B=0) == (0, b"") and call(T=0, table=0) == (0, b"")
        for bad in (dict(B=-1), dict(T=-1), dict(H=0), dict(Hkv=0), dict(D=0), dict(R=-2), dict(R=10), dict(table=-1)):
            assert call(**bad)[0] == -1 and b"bad size" in call(**bad)[1], bad
        assert call(Hkv=3)[0] == -1 and b"multiple" in call(Hkv=3)[1]
        assert call(R=3)[0] == -1 and b"even" in call(R=3)[1]
        assert call(dtype=7)[0] == -1 and call(table=2)[0] == -1 and b"tables" in call(table=2)[1]
        for bad in (dict(D=1 << 17), dict(B=1 << 31), dict(T=1 << 30, table=1 << 30), dict(B=1 << 20, T=1 << 20, table=1 << 20)):
            assert call(**bad)[0] == -2, bad
        for name in ("cos", "sin", "q", "k"):
            assert call(**{name: None})[0] == -1 and b"null" in call(**{name: None})[1], name
            assert call(**{name: ODD})[0] == -1 and b"aligned" in call(**{name: ODD})[1], name
        assert call(positions=ctypes.c_void_p(260), wide=1)[0] == -1
    assert back(P=0) == (0, b"") and back(P=-1)[0] == -1 and back(kv=3)[0] == -1 and back(g=None)[0] == -1 and back(v=None)[0] == -1
    assert forward(qkv=None)[0] == -1 and forward(qkv=ODD)[0] == -1


def test_gated_norm_statuses():
    lib = _lib.load()

    def at(n):
        return ctypes.c_void_p(n << 20)

    def forward(branch=at(1), residual=at(2), gate=at(3), w1=at(4), w2=at(5), normed=at(6), out=at(7), rows=4, dim=64, per=2, dtype=BF16, stream=F32, t1=BF16,
                t2=F32):
        return (lib.lbi_gated_residual_rmsnorm(branch, residual, gate, w1, w2, normed, out, rows, dim, per, 1e-5, 1.0, dtype, stream, t1, t2, None),
                lib.lbi_last_error())

    def back(g=at(1), branch=at(2), s=at(3), gs=at(4), gate=at(5), w1=at(6), w2=at(7), gb=at(8), gr=at(9), gg=at(10), g1=at(11), g2=at(12), ws=at(13),
             size=1 << 19, rows=4, dim=64, per=2, dtype=BF16, stream=F32, t1=BF16, t2=F32):
        return (lib.lbi_gated_residual_rmsnorm_pullback(g, branch, s, gs, gate, w1, w2, gb, gr, gg, g1, g2, ws, size, rows, dim, per, 1e-5, 1.0, dtype,
                                                        stream, t1, t2, None), lib.lbi_last_error())

    assert forward(rows=0) == (0, b"")
    for call in (forward, back):
        for bad in (dict(rows=-1), dict(dim=0), dict(per=-1), dict(per=3)):
            assert call(**bad)[0] == -1 and b"bad size" in call(**bad)[1], bad
        for bad in (dict(dtype=7), dict(stream=F16), dict(t1=F16), dict(t2=F16), dict(dtype=F32, stream=BF16)):
            assert call(**bad)[0] == -1 and b"bad dtype" in call(**bad)[1], bad
        for bad in (dict(dim=16385), dict(rows=1 << 31)):
            assert call(**bad)[0] == -2, bad
        for name in ("branch", "w1", "w2"):
            assert call(**{name: None})[0] == -1 and b"null" in call(**{name: None})[1], name
        for name in ("branch", "gate", "w1", "w2"):
            assert call(**{name: ODD})[0] == -1 and b"aligned" in call(**{name: ODD})[1], name
    for name in ("residual", "normed", "out"):
        assert forward(**{name: None})[0] == -1 and forward(**{name: ODD})[0] == -1, name
    for name in ("g", "s", "gb", "gr", "g1", "g2"):
        assert back(**{name: None})[0] == -1 and back(**{name: ODD})[0] == -1, name
    assert back(gg=None)[0] == -1 and back(gs=ODD)[0] == -1
    # overlaps: results on results, on inputs, on a part of their own
    near = ctypes.c_void_p((1 << 20) + 8)
    for bad in (dict(normed=near), dict(out=near), dict(normed=at(7)), dict(normed=at(3)), dict(out=at(4)), dict(out=at(5))):
        assert forward(**bad)[0] == -1 and b"overlaps" in forward(**bad)[1], bad
    for bad in (dict(gb=at(1)), dict(gr=at(3)), dict(gb=at(9)), dict(gg=at(5)), dict(g1=at(12)), dict(ws=at(2)), dict(g2=at(7))):
        assert back(**bad)[0] == -1 and b"overlaps" in back(**bad)[1], bad
    need = lib.lbi_gated_residual_rmsnorm_pullback_workspace_bytes(4, 64, 2)
    assert need >= 3 * 64 * 4 * 2 and back(size=need - 1)[0] == -4 and back(ws=None)[0] == -4
    for sizes in ((0, 64, 2), (4, 0, 2), (4, 64, 3), (4, 16385, 2), (4, 64, -1), (-4, 64, 2)):
        assert lib.lbi_gated_residual_rmsnorm_pullback_workspace_bytes(*sizes) == 0, sizes


def _call(**changed):
    base = dict(B=2, P=1, H=4, Hkv=2, T=100, Dk=64, Dv=64, q=256, k=256, v=256, q_stride=(25600, 6400, 64), k_stride=(12800, 6400, 64),
                v_stride=(12800, 6400, 64), log_decay=256, out=256, out_stride=(25600, 64, 256), state_out=256, g_out=256,
                g_out_stride=(25600, 25600, 6400, 64), dq=256, dk=256, dv=256, scale=1.0, dtype=BF16)
    return _lib.LinearAttentionCall(**{**base, **changed})


def test_linear_attention_statuses():
    lib = _lib.load()

    def run(entry, ws=OK, size=1 << 40, **changed):
        return getattr(lib, entry)(ctypes.byref(_call(**changed)), ws, size, None), lib.lbi_last_error()

    for entry in ("lbi_linear_attention", "lbi_linear_attention_pullback"):
        assert getattr(lib, entry)(None, None, 0, None) == -1
        assert run(entry, B=0) == (0, b"")
        for bad in (dict(B=-1), dict(H=0), dict(Hkv=0), dict(T=-1), dict(Dk=0), dict(Dv=0)):
            assert run(entry, **bad)[0] == -1 and b"bad size" in run(entry, **bad)[1], bad
        assert run(entry, Hkv=3)[0] == -1 and run(entry, dtype=F32)[0] == -2 and run(entry, dtype=9)[0] == -1
        for bad in (dict(Dk=129), dict(Dv=129), dict(T=1 << 30), dict(B=1 << 20), dict(B=1 << 19, H=512, Hkv=2)):
            assert run(entry, **bad)[0] == -2, bad
        for bad in (0.0, math.nan, math.inf):
            assert run(entry, scale=bad)[0] == -1 and b"scale" in run(entry, scale=bad)[1]
        for name in ("q", "k", "v", "log_decay"):
            assert run(entry, **{name: None})[0] == -1 and b"null" in run(entry, **{name: None})[1], name
            assert run(entry, **{name: 257})[0] == -1 and b"aligned" in run(entry, **{name: 257})[1], name
        assert run(entry, lengths=260, lengths_wide=1)[0] == -1 and run(entry, state=258)[0] == -1
        # few long chains are cut: their states go to the workspace
        need = getattr(lib, entry + "_workspace_bytes")(ctypes.byref(_call(B=1, T=8192)))
        assert need >= 2 * 4 * 64 * 64 * 4
        assert run(entry, B=1, T=8192, size=need - 1)[0] == -4 and run(entry, B=1, T=8192, ws=None)[0] == -4 and run(entry, B=1, T=8192, ws=ctypes.c_void_p(258))[0] == -1
        assert getattr(lib, entry + "_workspace_bytes")(ctypes.byref(_call(B=1, T=8192, Dk=200))) == 0
    assert run("lbi_linear_attention", out=None)[0] == -1 and run("lbi_linear_attention", state_out=257)[0] == -1
    pull = "lbi_linear_attention_pullback"
    assert run(pull, P=0) == (0, b"") and run(pull, P=-1)[0] == -1 and run(pull, P=1 << 20)[0] == -2
    for name in ("g_out", "dq", "dk", "dv"):
        assert run(pull, **{name: None})[0] == -1 and run(pull, **{name: 257})[0] == -1, name
    assert run(pull, g_state=258)[0] == -1 and run(pull, d_state=258)[0] == -1


def test_step_statuses():
    lib = _lib.load()

    def call(q=OK, k=OK, v=OK, l=OK, s=OK, active=None, out=OK, B=2, H=4, Hkv=2, Dk=64, Dv=64, dtype=BF16):
        return lib.lbi_linear_attention_step(q, k, v, l, s, active, out, B, H, Hkv, Dk, Dv, 1.0, dtype, None), lib.lbi_last_error()

    assert call(B=0) == (0, b"")
    for bad in (dict(B=-1), dict(H=0), dict(Hkv=0), dict(Dk=0), dict(Dv=0), dict(Hkv=3), dict(dtype=9)):
        assert call(**bad)[0] == -1, bad
    for bad in (dict(Dk=129), dict(Dv=129), dict(B=1 << 24)):
        assert call(**bad)[0] == -2, bad
    for name in ("q", "k", "v", "l", "s", "out"):
        assert call(**{name: None})[0] == -1 and call(**{name: ODD})[0] == -1, name


def test_wrappers_refuse_before_touching_a_device():
    h = torch.bfloat16
    q, k, v = torch.zeros(2, 4, 5, 8, dtype=h), torch.zeros(2, 2, 5, 8, dtype=h), torch.zeros(2, 2, 5, 6, dtype=h)
    l, s = torch.zeros(4), torch.zeros(2, 4, 8, 6)
    g = torch.zeros(2, 3, 4, 5, 6, dtype=h)
    for bad in ((q[0], k, v), (q, k[..., :4], v), (q, k, v[:, :1]), (q, k[:1], v[:1]), (q, k[:, :, :4], v[:, :, :4])):
        with pytest.raises(ValueError, match="must be"):
            mixer.linear_attention(*bad, l, scale=1.0)
    with pytest.raises(ValueError, match="multiple"):
        mixer.linear_attention(q[:, :3], k, v, l[:3], scale=1.0)
    for call in (lambda **m: mixer.linear_attention(q, k, v, m.pop("l", l), scale=m.pop("scale", 1.0), **m),
                 lambda **m: mixer.linear_attention_input_pullback_basis(q, k, v, g, m.pop("l", l), scale=m.pop("scale", 1.0), **m)):
        for bad in (dict(l=l[:2]), dict(l=l.double()), dict(scale=0.0), dict(scale=math.nan), dict(state=s.half()), dict(state=s[:, :2]),
                    dict(lengths=torch.zeros(2)), dict(lengths=torch.zeros(3, dtype=torch.int32))):
            with pytest.raises(ValueError):
                call(**bad)
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        mixer.linear_attention(q.float(), k.float(), v.float(), l, scale=1.0)
    with pytest.raises(ValueError, match="one dtype"):
        mixer.linear_attention(q, k.half(), v, l, scale=1.0)
    for bad in (g[0], g[:, :, :2], g.half(), g[..., :4]):
        with pytest.raises(ValueError, match="basis"):
            mixer.linear_attention_input_pullback_basis(q, k, v, bad, l, scale=1.0)
    with pytest.raises(ValueError, match="g_state"):
        mixer.linear_attention_input_pullback_basis(q, k, v, g, l, scale=1.0, g_state=s)
    token = q[:, :, 0], k[:, :, 0], v[:, :, 0]
    for bad in (s.half(), s[:, :2], torch.zeros(2, 4, 6, 8).mT):
        with pytest.raises(ValueError, match="state"):
            mixer.linear_attention_step(*token, l, bad, scale=1.0)
    with pytest.raises(ValueError, match="active"):
        mixer.linear_attention_step(*token, l, s, scale=1.0, active=torch.ones(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        mixer.linear_attention_step(*token, l, s, scale=1.0)

    qkv, cos = torch.zeros(2, 5, 8 * 8), torch.zeros(5, 4)
    heads = dict(n_heads=4, n_kv_heads=2)
    for bad in ((qkv[0], cos, cos), (qkv[..., :60], cos, cos), (qkv, cos[:4], cos[:4]), (qkv, cos, cos[:4]), (qkv, torch.zeros(5, 5), torch.zeros(5, 5)),
                (qkv, cos.half(), cos.half())):
        with pytest.raises(ValueError, match="rotary_heads"):
            mixer.rotary_heads(*bad, **heads)
    with pytest.raises(ValueError, match="divisible"):
        mixer.rotary_heads(qkv, cos, cos, n_heads=4, n_kv_heads=3)
    for bad in (torch.zeros(5), torch.zeros(4, dtype=torch.int64), torch.zeros(1, 5, dtype=torch.int64)):
        with pytest.raises(ValueError, match="positions"):
            mixer.rotary_heads(qkv, cos, cos, **heads, positions=bad)
    with pytest.raises(TypeError):
        mixer.rotary_heads(qkv.double(), cos, cos, **heads)
    with pytest.raises(RuntimeError, match="CUDA"):
        mixer.rotary_heads(qkv, cos, cos, **heads)
    dq = torch.zeros(2, 1, 4, 5, 8)
    for bad in ((dq[0], dq, dq), (dq, dq[:, :, :3], dq[:, :, :3]), (dq, dq, dq[..., :4]), (dq, dq.half(), dq), (dq, dq[:, :, :, :4], dq[:, :, :, :4])):
        with pytest.raises(ValueError):
            mixer.rotary_heads_pullback(*bad, cos, cos, n_kv_heads=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        mixer.rotary_heads_pullback(dq, dq, dq, cos, cos, n_kv_heads=2)

    x, w = torch.zeros(2, 3, 16), torch.ones(16)
    for bad in ((x, x[:1], w, w), (x, x, w[1:], w), (x, x, w, w[1:])):
        with pytest.raises(ValueError):
            block.gated_residual_rmsnorm(*bad, 1e-5)
    for bad in (w.half(), w[1:], torch.ones(2, 16), torch.ones(3, 1, 16), torch.ones(2, 3, 1), torch.ones(1, 1, 16)):
        with pytest.raises(ValueError, match="gate"):
            block.gated_residual_rmsnorm(x, x, w, w, 1e-5, gate=bad)
        with pytest.raises(ValueError, match="gate"):
            block.gated_residual_rmsnorm_pullback(x, x, x, w, w, 1e-5, gate=bad)
    with pytest.raises(ValueError, match="stream"):
        block._norm_types("stream", h, torch.float16, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        block.gated_residual_rmsnorm(x, x, w, w, 1e-5, gate=torch.ones(2, 1, 16))
    for bad in (dict(g_residual=x.half()), dict(g_residual=x[:1])):
        with pytest.raises(ValueError, match="g_residual"):
            block.gated_residual_rmsnorm_pullback(x, x, x, w, w, 1e-5, **bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        block.gated_residual_rmsnorm_pullback(x, x, x, w, w, 1e-5)


def test_rotary_tables():
    cos, sin = mixer.rotary_tables(200_000, 8, base=100.0, device="cpu", magnitude=1.5)
    for t, i in ((0, 0), (1, 3), (199_999, 0), (123_456, 2)):
        angle = t * 100.0 ** (-2 * i / 8)
        assert abs(float(cos[t, i]) - 1.5 * math.cos(angle)) < 1e-6 and abs(float(sin[t, i]) - 1.5 * math.sin(angle)) < 1e-6
    slow, _ = mixer.rotary_tables(100, 8, base=100.0, device="cpu", factor=4.0)
    assert torch.allclose(slow[4 * torch.arange(25)], mixer.rotary_tables(25, 8, base=100.0, device="cpu")[0], atol=1e-7)
    # of 64 elements over 1000 positions the fast ones turn more than 32 times and stay, the slowest less than once and are stretched eightfold
    plain, _ = mixer.rotary_tables(4000, 64, device="cpu")
    cos, _ = mixer.rotary_tables(4000, 64, device="cpu", factor=8.0, original_length=1000)
    turns = [1000 * 10000.0 ** (-2 * i / 64) / (2 * math.pi) for i in range(32)]
    for i, count in enumerate(turns):
        keep = min(max((count - 1.0) / 31.0, 0.0), 1.0)
        f = 10000.0 ** (-2 * i / 64) * (keep + (1 - keep) / 8)
        assert abs(float(cos[3999, i]) - math.cos(3999 * f)) < 1e-6, i
        assert (count < 32) or torch.equal(cos[:, i], plain[:, i])
    assert turns[0] > 32 and turns[-1] < 1
    for bad in (dict(length=-1), dict(rotary_dim=3), dict(base=0.0), dict(factor=0.0), dict(factor=math.inf), dict(original_length=0),
                dict(original_length=5, ramp=(2.0, 1.0)), dict(magnitude=math.nan)):
        with pytest.raises(ValueError, match="rotary_tables"):
            mixer.rotary_tables(**{**dict(length=4, rotary_dim=8, device="cpu"), **bad})


def test_a_step_refuses_a_state_that_shares_memory():
    lib = _lib.load()
    bsz, heads, shared, dim = 2, 4, 2, 64
    sizes = dict(state=bsz * heads * dim * dim * 4, out=bsz * heads * dim * 2, q=bsz * heads * dim * 2, k=bsz * shared * dim * 2,
                 v=bsz * shared * dim * 2, log_decay=heads * 4, active=bsz)
    place, at = {}, 1 << 20
    for name, size in sizes.items():
        place[name], at = at, at + (size + 255) // 256 * 256
    for written in ("state", "out"):
        for other in sizes:
            if other == written:
                continue
            for shift in (0, sizes[written] - 4, 4 - sizes[other] if sizes[other] >= 8 else 0):  # from the start, over the end, over the start
                p = {**place, other: (1 << 30) + shift, written: 1 << 30}
                status = lib.lbi_linear_attention_step(*(ctypes.c_void_p(p[n]) for n in ("q", "k", "v", "log_decay", "state", "active", "out")), bsz, heads,
                                                       shared, dim, dim, 1.0, BF16, None)
                assert status == -1 and b"overlaps" in lib.lbi_last_error(), (written, other, shift)
