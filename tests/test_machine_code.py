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


def _scalars(operand: str) -> range:
    m = re.match(r"s(?:\[(\d+):(\d+)\]|(\d+))$", operand)
    if m is None:
        return range(0)
    return range(int(m[3]), int(m[3]) + 1) if m[3] else range(int(m[1]), int(m[2]) + 1)


def test_scalars_from_vector_instructions_reach_memory_instructions_in_time(listings):
    """A scalar register that a vector instruction has written (a spilled one that comes back by v_readlane, a v_readfirstlane) may be read by a memory instruction
    five wait states later at the earliest.  The compiler sees to it, but not for memory instructions in inline assembly."""
    memory, found = ("buffer_", "global_", "scratch_", "flat_"), 0
    from_vector = re.compile(r"^\s*v_read(?:first)?lane_b32 s(\d+), .*$", re.M)
    for listing in listings:
        text = listing.read_text()
        for m in from_vector.finditer(text):
            found += 1
            register, states, at = int(m[1]), 0, m.end() + 1
            while states < 5 and at < len(text):
                end = text.find("\n", at)
                line = text[at:end].split("//")[0].strip()
                at = end + 1
                if line.endswith(":"):
                    continue
                op, _, rest = line.partition(" ")
                if op in ("", "s_endpgm"):
                    break
                operands = [part.split(" ")[0] for part in re.split(r",\s*", rest)]
                if op.startswith(memory):
                    assert not any(register in _scalars(operand) for operand in operands), (m[0].strip(), line, text[m.start():end])
                elif op.startswith("s_") and register in _scalars(operands[0]) and not op.startswith("s_cmp"):
                    break  # a scalar instruction's result is there at once
                states += int(operands[0], 0) + 1 if op == "s_nop" else 1
    assert found > 1000


def test_linear_attentions_waits_count_stores_that_are_there(listings):
    """At a chunk's end the kernel waits until all but its last four memory operations are done: the results' four stores, behind which the next tiles were asked
    for before.  Whole chunks and a last one have their own."""
    seen = 0
    for listing in listings:
        if b"linear_attn12chunk_kernel" not in listing.read_bytes():
            continue
        for symbol, body in _kernels(listing):
            m = re.search(r"chunk_kernelI\w+?Li(\d+)ELi(\d+)ELb(\d)ELb(\d)ELi\dELb(\d)E", symbol)
            if m is None or m.groups()[2:] != ("1", "1", "0"):
                continue
            seen += 1
            width = 4 if m[2] == "128" else 2
            stores = len(re.findall(rf"^\s*buffer_store_dwordx{width} ", body, re.M))
            assert stores == 8, (symbol, stores)
    assert seen == 12  # four widths, three of types and planes
