"""What the entry points of the block's MLP half and of the clipping refuse, each with its status and before anything is launched; and
what their Python wrappers refuse without a device."""
from __future__ import annotations

import ctypes

import pytest
import torch

from latent_bounded_interfaces_amd import _lib

OK, ODD = ctypes.c_void_p(256), ctypes.c_void_p(257)  # never dereferenced
F32, F16, BF16 = _lib.LBI_F32, _lib.LBI_F16, _lib.LBI_BF16


def test_norm_statuses():
    lib = _lib.load()

    def call(hidden=OK, residual=OK, weight=OK, normed=OK, out=OK, scales=None, rows=4, dim=64, dtype=BF16, stream=F32, w=BF16):
        return lib.lbi_residual_rmsnorm(hidden, residual, weight, normed, out, scales, rows, dim, 1e-5, dtype, stream, w, None), lib.lbi_last_error()

    assert call(rows=0) == (0, b"") and call(rows=0, hidden=None) == (0, b"")
    for bad in (dict(rows=-1), dict(dim=0), dict(dim=-8)):
        assert call(**bad)[0] == -1 and b"bad size" in call(**bad)[1], bad
    for bad in (dict(dtype=7), dict(dtype=-1), dict(stream=F16), dict(dtype=F32, stream=BF16), dict(w=F16), dict(dtype=F32, w=BF16)):
        assert call(**bad)[0] == -1 and b"bad dtype" in call(**bad)[1], bad
    for bad in (dict(dim=16385), dict(rows=1 << 31)):
        assert call(**bad)[0] == -2, bad
    for name in ("hidden", "weight", "normed"):
        assert call(**{name: None})[0] == -1 and b"null" in call(**{name: None})[1]
    for name in ("hidden", "residual", "weight", "normed", "out", "scales"):
        assert call(**{name: ODD})[0] == -1 and b"aligned" in call(**{name: ODD})[1], name


def test_norm_pullback_statuses():
    lib = _lib.load()

    def call(g=OK, s=OK, gs=OK, weight=OK, gh=OK, gr=OK, gw=OK, ws=OK, size=1 << 40, rows=4, dim=64, dtype=BF16, stream=F32, w=BF16):
        return lib.lbi_residual_rmsnorm_pullback(g, s, gs, weight, gh, gr, gw, ws, size, rows, dim, 1e-5, dtype, stream, w, None), lib.lbi_last_error()

    need = lib.lbi_residual_rmsnorm_pullback_workspace_bytes(4, 64)
    assert need > 0 and need % (64 * 4) == 0
    assert lib.lbi_residual_rmsnorm_pullback_workspace_bytes(0, 64) == 0
    assert lib.lbi_residual_rmsnorm_pullback_workspace_bytes(4, 0) == 0 and lib.lbi_residual_rmsnorm_pullback_workspace_bytes(1 << 31, 64) == 0
    assert call(size=need - 1)[0] == -4 and call(ws=None)[0] == -4
    for bad in (dict(rows=-1), dict(dim=0), dict(dtype=7), dict(stream=F16), dict(w=F16), dict(gw=None), dict(g=None), dict(s=None),
                dict(weight=None), dict(gh=None, gr=None), dict(rows=0, gw=None)):
        assert call(**bad)[0] == -1, bad
    assert call(dim=16385)[0] == -2
    for name in ("g", "s", "gs", "weight", "gh", "gr", "gw", "ws"):
        assert call(**{name: ODD})[0] == -1 and b"aligned" in call(**{name: ODD})[1], name


def test_mlp_statuses():
    lib = _lib.load()
    eight = ctypes.c_void_p(264)

    def forward(x=OK, w1=OK, b1=OK, w2=OK, b2=OK, z=OK, a=OK, out=OK, ws=OK, size=1 << 40, rows=16, dim=64, hidden=64, width=64, dtype=BF16):
        return lib.lbi_gated_mlp(x, w1, b1, w2, b2, z, a, out, ws, size, rows, dim, hidden, width, dtype, None), lib.lbi_last_error()

    def pullback(g=OK, x=OK, z=OK, a=OK, w1=OK, w2=OK, gx=OK, g1=OK, g2=OK, gb1=OK, gb2=OK, ws=OK, size=1 << 40, rows=16, dim=64, hidden=64,
                 width=64, dtype=BF16):
        return (lib.lbi_gated_mlp_vjp(g, x, z, a, w1, w2, gx, g1, g2, gb1, gb2, ws, size, rows, dim, hidden, width, dtype, None),
                lib.lbi_last_error())

    assert forward(rows=0) == (0, b"") and pullback(rows=0)[0] == -2
    for call in (forward, pullback):
        for bad in (dict(rows=-1), dict(dim=-8), dict(hidden=-8), dict(width=-8), dict(dim=0), dict(hidden=0), dict(width=0)):
            assert call(**bad)[0] == -1 and b"bad size" in call(**bad)[1], bad
        for bad in (dict(dtype=F32), dict(dtype=7), dict(dim=(1 << 20) + 8), dict(rows=(1 << 23) + 1)):
            assert call(**bad)[0] == -2, bad
    for name in ("x", "w1", "w2", "a", "out"):
        assert forward(**{name: None})[0] == -1 and b"null" in forward(**{name: None})[1]
    for name in ("x", "w1", "b1", "w2", "b2", "z", "a", "out", "ws"):
        assert forward(**{name: eight})[0] == -1 and b"aligned" in forward(**{name: eight})[1], name
    for name in ("g", "x", "z", "a", "w1", "w2", "gx", "g1", "g2"):
        assert pullback(**{name: None})[0] == -1 and b"null" in pullback(**{name: None})[1]
    for name in ("g", "x", "z", "a", "w1", "w2", "gx", "g1", "g2", "gb1", "gb2", "ws"):
        assert pullback(**{name: eight})[0] == -1 and b"aligned" in pullback(**{name: eight})[1], name
    need = lib.lbi_gated_mlp_vjp_workspace_bytes(16, 64, 64, 64)
    assert need >= 16 * 128 * 2 and pullback(size=need - 1)[0] == -4 and pullback(ws=None)[0] == -4
    # long sums of few results are cut: the parts go to the workspace
    need = lib.lbi_gated_mlp_workspace_bytes(64, 256, 8192, 256)
    assert need > 0
    big = dict(rows=64, dim=256, hidden=8192, width=256)
    assert forward(**big, size=need - 1)[0] == -4 and forward(**big, ws=None)[0] == -4
    # widths that are padded: the copies too
    assert lib.lbi_gated_mlp_workspace_bytes(16, 63, 64, 64) >= 2 * (16 * 64 + 128 * 64) and forward(dim=63, ws=None)[0] == -4
    for sizes in ((0, 64, 64, 64), (16, 0, 64, 64), (-1, 64, 64, 64)):
        assert lib.lbi_gated_mlp_workspace_bytes(*sizes) == 0 and lib.lbi_gated_mlp_vjp_workspace_bytes(*sizes) == 0


def test_clip_statuses():
    lib = _lib.load()

    def call(*rows, n=None, max_norm=1.0, norm=OK, ws=OK, size=1 << 40, empty=False):
        words = [w for row in rows for w in row]
        table = None if empty else (ctypes.c_int64 * max(len(words), 1))(*words)
        return lib.lbi_clip_gradients(table, len(rows) if n is None else n, max_norm, norm, ws, size, None), lib.lbi_last_error()

    a, b = (4096, 8192, 100, F32), (16384, 20480, 100, BF16)
    need = lib.lbi_clip_gradients_workspace_bytes(2)
    assert need > 0 and lib.lbi_clip_gradients_workspace_bytes(1000) > need and lib.lbi_clip_gradients_workspace_bytes(-1) > 0
    assert call(a, b, size=need - 1)[0] == -4 and call(a, b, ws=None)[0] == -4
    assert call(a, b, n=-1)[0] == -1 and call(n=3, empty=True)[0] == -1
    for bad in ((4096, 8192, -1, F32), (4096, 8192, 100, 3), (4096, 8192, 100, -1), (0, 8192, 100, F32), (4098, 8192, 100, F32),
                (4096, 8194, 100, F32), (4097, 8192, 100, BF16), (4096, 8192, 1 << 41, F32)):
        assert call(bad)[0] == -1, bad
    assert call((4096, 0, 1 << 39, F32), (4096, 0, (1 << 39) + 1, F32))[0] == -1
    for bad in (-1.0, float("nan")):
        assert call(a, b, max_norm=bad)[0] == -1 and b"max_norm" in call(a, b, max_norm=bad)[1]
    assert call(a, b, norm=None)[0] == -1 and call(a, b, norm=ctypes.c_void_p(258))[0] == -1 and call(a, b, ws=ctypes.c_void_p(260))[0] == -1
    # results on results, on other inputs, on a part of their own
    for bad in ([a, (16384, 8192, 100, BF16)], [a, (16384, 8192 + 396, 1, F32)], [a, (8192, 20480, 100, BF16)], [(4096, 4100, 100, F32)],
                [(4096, 4096, 100, F32), (4096, 4096, 100, F32)], [(4096, 8192, 100, F32), (8192, 4096, 100, F32)],
                [(4096, 8192, 100, F32), (16384, 4096, 100, F32)]):
        assert call(*bad)[0] == -1 and b"overlaps" in call(*bad)[1], bad


def test_wrappers_refuse_before_touching_a_device():
    from latent_bounded_interfaces_amd.hip.gradients import clip_gradients, gradient_norm
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp, residual_rmsnorm, residual_rmsnorm_pullback

    x, w = torch.zeros(4, 16), torch.ones(16)
    with pytest.raises(ValueError, match="shaped like hidden"):
        residual_rmsnorm(x, x[:2], w, 1e-5)
    with pytest.raises(ValueError, match="weight"):
        residual_rmsnorm(x, x, w[1:], 1e-5)
    with pytest.raises(RuntimeError, match="CUDA"):
        residual_rmsnorm(x, x, w, 1e-5)
    with pytest.raises(ValueError, match="weight"):
        residual_rmsnorm_pullback(x, x, w[1:], 1e-5)
    with pytest.raises(ValueError, match="g_residual"):
        residual_rmsnorm_pullback(x, x, w, 1e-5, g_residual=x.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        residual_rmsnorm_pullback(x, x, w, 1e-5)
    fc1, fc2 = torch.zeros(48, 16, dtype=torch.bfloat16), torch.zeros(8, 24, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        gated_mlp(x, fc1, fc2)
    x = x.bfloat16()
    for bad in ((fc1[:46], fc2), (fc1, fc2[:, :20]), (fc1.view(-1), fc2), (fc1[:, :8], fc2)):
        with pytest.raises(ValueError, match="gated_mlp"):
            gated_mlp(x, *bad)
    with pytest.raises(ValueError, match="widths"):
        gated_mlp(x, fc1, fc2[:0])
    with pytest.raises(ValueError, match="fc1_bias"):
        gated_mlp(x, fc1, fc2, torch.zeros(24))
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_mlp(x, fc1, fc2)
    g, z, a = torch.zeros(4, 8).bfloat16(), torch.zeros(4, 48).bfloat16(), torch.zeros(4, 24).bfloat16()
    for bad in ((g[:, :4], x, z, a), (g, x, z[:2], a), (g, x, z, a.half()), (g.float(), x, z, a)):
        with pytest.raises(ValueError, match="gated_mlp_vjp"):
            gated_mlp_vjp(*bad, fc1, fc2)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_mlp_vjp(g, x, z, a, fc1, fc2)
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_gradients([w], 1.0)
    with pytest.raises(TypeError):
        gradient_norm([1.0])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_gradients([w], bad)
    with pytest.raises(ValueError, match="one tensor"):
        clip_gradients([w], 1.0, out=[])
    assert gradient_norm([]).item() == 0.0


def test_clipping_that_is_refused_leaves_no_gradients_behind():
    from latent_bounded_interfaces_amd.backward import ScanADEngine, assign_clipped_grad_map

    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_grad_norm"):
            ScanADEngine(max_grad_norm=bad)
    layer = torch.nn.Linear(3, 2)
    layer.weight.grad = torch.ones(2, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        assign_clipped_grad_map(layer, {"weight": torch.ones(2, 3), "bias": torch.ones(2)}, 1.0)
    assert layer.weight.grad is None and layer.bias.grad is None
