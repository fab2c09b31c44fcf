"""What the kernels' own waits rest on, looked up in the machine code of the built library: the compiler knows nothing of what inline assembly and counted waits
need, and may merge, move or spill what they count on."""
from __future__ import annotations

import os
import re
import shutil
import struct
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

from latent_bounded_interfaces_amd import _lib

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _objdump() -> str | None:
    places = (os.environ.get("ROCM_PATH", "/opt/rocm"), "/opt/rocm")
    return next((str(p) for p in (Path(place) / "llvm" / "bin" / "llvm-objdump" for place in places) if p.exists()), shutil.which("llvm-objdump"))


def _code_objects() -> list[bytes]:
    data, found = _lib.LIB_PATH.read_bytes(), []
    at = data.find(MAGIC)
    while at >= 0:
        (count,), place = struct.unpack_from("<Q", data, at + 24), at + 32
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, place)
            if size and b"gfx950" in data[place + 24:place + 24 + name]:
                found.append(data[at + offset:at + offset + size])
            place += 24 + name
        at = data.find(MAGIC, at + len(MAGIC))
    return found


@pytest.fixture(scope="module")
def listings(tmp_path_factory) -> list[Path]:
    """The instructions of each code object, a file each."""
    objdump = _objdump()
    if objdump is None:
        pytest.skip("no llvm-objdump")
    _lib.load()  # (says so if there is no library)
    folder = tmp_path_factory.mktemp("code")

    def listing(item) -> Path:
        number, code = item
        of, to = folder / f"{number}.o", folder / f"{number}.txt"
        of.write_bytes(code)
        with open(to, "wb") as out:
            subprocess.run([objdump, "-d", "--no-show-raw-insn", "--no-leading-addr", str(of)], stdout=out, check=True)
        of.unlink()
        return to

    with ThreadPoolExecutor(4) as pool:
        files = list(pool.map(listing, enumerate(_code_objects())))
    assert files
    yield files
    shutil.rmtree(folder)


def _kernels(listing: Path):
    """(symbol, its lines)"""
    for part in re.split(r"\n(?=<)", listing.read_text()):
        head, _, body = part.partition("\n")
        if head.startswith("<"):
            yield head.strip("<>: "), body


def test_the_narrow_scans_first_waits_count_stores_that_are_there(listings):
    """A step's waits count the stores of the steps before it.  The first steps have none, so the kernel issues as many into nothing; fewer, and a wait would let
    rows be read that are still on their way."""
    seen = 0
    for listing in listings:
        if b"scan_narrow_kernel" not in listing.read_bytes():
            continue
        for symbol, body in _kernels(listing):
            m = re.search(r"scan_narrow_kernelI\w+?Li(\d+)ELi(\d+)ELb\dELi(\d+)E", symbol)
            if m is None or int(m[3]) == 0:
                continue
            seen += 1
            stores = len(re.findall(r"^\s*buffer_store_dword v\d+, off, s\[\d+:\d+\], 0\s*(?://.*)?$", body, re.M))
            assert stores >= 4 * int(m[2]) * int(m[3]), (symbol, stores)
    assert seen >= 20
