"""What the entry points of the block's MLP half and of the clipping refuse beside what their own tests name, without a device."""
from __future__ import annotations

import ctypes

from latent_bounded_interfaces_amd import _lib

F32, F16, BF16 = _lib.LBI_F32, _lib.LBI_F16, _lib.LBI_BF16


def test_norm_results_that_lie_on_other_tensors():
    """4 rows of 64: 512 bytes in bf16, 1024 in fp32, 256 in 8 bits.  Addresses that are never dereferenced."""
    lib = _lib.load()

    def forward(hidden=4096, residual=8192, normed=12288, out=16384, scales=None, stream=F32):
        return lib.lbi_residual_rmsnorm(hidden, residual, 256, normed, out, scales, 4, 64, 1e-5, BF16, stream, BF16, None), lib.lbi_last_error()

    for bad in (dict(normed=4096 + 256), dict(normed=4096 - 256), dict(normed=8192), dict(out=4096), dict(out=8192 + 512), dict(out=12288),
                dict(out=12288 - 512), dict(normed=4096, scales=512), dict(normed=8192 + 768, scales=512), dict(normed=16384 + 768, scales=512),
                dict(normed=4096, out=4096, stream=BF16), dict(out=4096 + 256, stream=BF16)):
        assert forward(**bad)[0] == -1 and b"overlaps" in forward(**bad)[1], bad

    def pullback(g=4096, s=8192, more=12288, gh=16384, gr=20480, stream=F32):
        return (lib.lbi_residual_rmsnorm_pullback(g, s, more, 256, gh, gr, 512, 1024, 1 << 40, 4, 64, 1e-5, BF16, stream, BF16, None),
                lib.lbi_last_error())

    for bad in (dict(gh=4096 + 256), dict(gh=8192), dict(gh=12288 + 512), dict(gr=4096), dict(gr=8192 + 512), dict(gr=12288 - 512),
                dict(gh=20480), dict(gh=20480 + 768), dict(gh=20480 + 256, stream=BF16)):
        assert pullback(**bad)[0] == -1 and b"overlaps" in pullback(**bad)[1], bad
