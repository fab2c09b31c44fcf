"""The gated MLP in every layout that its products take: which those are, by the arithmetic that chooses them, and results in whole numbers,
which no order of sums and no cut changes and in which a single missing term shows."""
from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / "latent_bounded_interfaces_amd" / "csrc"
U = 2.0 ** -24

#: (rows, D, hidden, width).  Between them the five products (gated, down, its cotangent, the input's, both weights') take each tile that they take on 256 compute
#: units, with all sums whole, with all cut into parts, and with whole rounds followed by cut tiles: 88 combinations, of which the sizes of
#: test_block_gpu.py reach 49.
MLP_LAYOUTS = [
    (2, 5255, 295, 5935), (646, 53, 19, 5949), (961, 5819, 16, 107), (962, 854, 25, 5915), (125, 5570, 961, 5115), (2440, 55, 18, 5593),
    (131, 5886, 2395, 275), (2330, 2, 1673, 6), (3424, 5410, 67, 1), (3350, 175, 170, 2867), (866, 4915, 1244, 43), (609, 5291, 2103, 13),
    (1263, 5674, 1067, 42), (1855, 2, 3205, 517), (1397, 4789, 1249, 222), (200, 1135, 4364, 5454), (1191, 3152, 2352, 31),
    (1516, 37, 1325, 5206), (1558, 3681, 1660, 257), (605, 2882, 4306, 24), (1127, 5449, 1981, 37), (2429, 3376, 1460, 3), (4146, 5997, 449, 57),
    (4204, 648, 2990, 25), (1035, 122, 3000, 5438), (908, 4118, 4080, 63), (2186, 50, 5399, 964), (1747, 1611, 4985, 19), (196, 4555, 9561, 217),
    (6442, 1, 7069, 1), (1054, 4, 3461, 5548), (1211, 4895, 3504, 36), (7823, 50, 617, 3091), (1423, 39, 3034, 5448), (2332, 16, 2522, 4042),
    (6587, 2760, 1239, 16), (11675, 1167, 1093, 3), (2399, 62, 3427, 3485), (1349, 4652, 4968, 2), (3724, 11, 1543, 5901), (3523, 4, 2957, 5253),
    (1319, 222, 11219, 3023), (13775, 46, 563, 5883), (1409, 5, 9902, 5245), (6608, 27, 2728, 4550)]

HOST = """
#include <initializer_list>
#include "lbi_block_mlp_layout.h"
using namespace lbi::block_mlp;
extern "C" void layouts(int64_t rows, int64_t D, int64_t hidden, int64_t width, int* out) {
    for (int64_t* n : {&D, &hidden, &width}) *n = (*n + 7) / 8 * 8;
    const Layout all[5] = {layout_of(256, rows, hidden, D, GATED, 0), layout_of(256, rows, width, hidden, PLAIN, 0),
                           layout_of(256, rows, hidden, width, UNGATED, 1), layout_of(256, rows, D, 2 * hidden, PLAIN, 1),
                           layout_of(256, 2 * hidden, D, rows, PLAIN, 2, width, hidden)};
    for (int i = 0; i < 5; ++i) out[2 * i] = all[i].form, out[2 * i + 1] = all[i].parts == 1 ? 0 : all[i].whole ? 2 : 1;
}
"""


@pytest.fixture(scope="module")
def layouts(tmp_path_factory):
    """(rows, D, hidden, width) -> {(product, tile, whole / cut / both)}."""
    compiler = shutil.which("g++") or shutil.which("clang++") or "/opt/rocm/llvm/bin/clang++"
    folder = tmp_path_factory.mktemp("layouts")
    (folder / "host.cpp").write_text(HOST)
    subprocess.run([compiler, "-O2", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(folder / "host.cpp"), "-o", str(folder / "host.so")], check=True)
    call = ctypes.CDLL(str(folder / "host.so")).layouts
    call.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_void_p]
    out = (ctypes.c_int * 10)()

    def of(sizes):
        call(*sizes, out)
        return {(i, out[2 * i], out[2 * i + 1]) for i in range(5)}

    return of


def test_every_layout_is_among_the_sizes(layouts):
    covered = set().union(*map(layouts, MLP_LAYOUTS))
    # whole rounds followed by cut tiles: tiles of 256 x 256 for every product, the pair of weights' gradients among them
    assert {(product, 0, 2) for product in range(4)} <= covered and (4, 1, 2) in covered
    rng = random.Random(1)

    def spread(low, high):
        return max(low, min(high, round(low * (high / low) ** rng.random())))

    reached = 0
    for _ in range(60_000):
        rows, dim, hidden = spread(1, 16384), spread(16, 6000), spread(16, 12000)
        width = dim if rng.random() < 0.5 else spread(16, 6000)
        if rows * hidden * max(dim, width) <= 150_000_000_000:
            reached += 1
            new = layouts((rows, dim, hidden, width)) - covered
            assert not new, f"{(rows, dim, hidden, width)} takes {new}, which none of the sizes does"
    assert reached > 50_000


def _few(gen, *shape, share):
    """-1, 0 and 1, that many of them not 0."""
    some = torch.rand(*shape, generator=gen, device="cuda") < share
    return some * (2.0 * torch.randint(0, 2, shape, generator=gen, device="cuda") - 1.0)


def _share(most, terms):
    return min(1.0, most / terms)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,hidden,width", MLP_LAYOUTS)
def test_mlp_in_whole_numbers(rows, dim, hidden, width, dtype, device):
    from latent_bounded_interfaces_amd.hip.transformer.block import gated_mlp, gated_mlp_vjp

    gen = torch.Generator(device="cuda").manual_seed(rows + dim)
    half = torch.finfo(dtype).eps / 2

    def near(got, value, error):
        bound = error * (1 + half) + half * value.abs() + torch.finfo(dtype).smallest_normal * half
        assert bool(((got.double() - value).abs() <= bound).all())

    # forwards: up and gate are whole numbers, each product is held against what the kernels themselves put into it
    x, fc1 = (_few(gen, *shape, share=_share(4, dim) ** 0.5).to(dtype) for shape in ((rows, dim), (2 * hidden, dim)))
    fc2, b1, b2 = (_few(gen, *shape, share=0.5).to(dtype) for shape in ((width, hidden), (2 * hidden,), (width,)))
    out, z, a = gated_mlp(x, fc1, fc2, b1, b2, keep=True)
    assert torch.equal(gated_mlp(x, fc1, fc2, b1, b2), out)
    want = x.double() @ fc1.double().t() + b1.double()
    assert torch.equal(z, want.to(dtype))
    up, gate = want.chunk(2, -1)
    want = up * gate * torch.sigmoid(gate)
    near(a, want, (gate.abs() + 6) * 2 * U * want.abs())  # exp and the division that make the sigmoid, two products
    size = a.double().abs() @ fc2.double().abs().t() + b2.double().abs()
    near(out, a.double() @ fc2.double().t() + b2.double(), (hidden + 2) * 2 * U * size)
    # backwards: gates at which the activation and its derivative are whole numbers (silu(0) = 0 with slope 1/2, silu(64) = 64 with slope 1 and
    # silu(-200) = 0 with slope 0 in fp32), so that the cotangent of fc1_output is too; up's weights are 64ths
    gate = torch.tensor([0.0, 64.0, -200.0], device=device)[torch.randint(0, 3, (rows, hidden), generator=gen, device=device)]
    up = torch.where(gate == 0, 2.0, 1.0) * _few(gen, rows, hidden, share=1.0)
    g_out, fc2 = (_few(gen, *shape, share=_share(4, width) ** 0.5) for shape in ((rows, width), (width, hidden)))
    x, a = (_few(gen, rows, n, share=_share(100, rows)) for n in (dim, hidden))
    fc1 = _few(gen, 2 * hidden, dim, share=_share(100, hidden))
    fc1[:hidden] /= 64
    got = gated_mlp_vjp(*(t.to(dtype) for t in (g_out, x, torch.cat((up, gate), -1), a, fc1, fc2)), bias=True)
    g_out, x, a, fc1, fc2 = (t.double() for t in (g_out, x, a, fc1, fc2))
    g_a = g_out @ fc2
    g_z = torch.cat((g_a * gate.clamp_min(0), g_a * torch.where(gate == 0, up / 2, torch.where(gate > 0, up, 0.0))), -1)
    assert torch.equal(g_z.to(dtype).double(), g_z)
    for one, want in zip(got, (g_z @ fc1, g_z.t() @ x, g_out.t() @ a, g_z.sum(0), g_out.sum(0))):
        assert torch.equal(one, want.to(dtype))
