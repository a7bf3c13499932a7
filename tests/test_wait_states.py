"""The wait states of the built kernels' memory instructions, read from the library's own disassembly: a vector memory
instruction may read a scalar register (its buffer resource, its offset) five wait states after a vector instruction
wrote it (v_readfirstlane and the like) and no earlier. The compiler keeps that distance for the instructions that it
forms; for those written in inline assembly the assembly has to."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

LIB = Path(__file__).resolve().parents[1] / "zonos3-mini_amd" / "lib" / "libzonos3_gdn.so"
NEEDED = 5
MEMORY = ("buffer_", "global_", "flat_", "scratch_")


def _objdump() -> str:
    near = Path(shutil.which("hipcc") or "/opt/rocm/bin/hipcc").resolve().parents[1] / "llvm" / "bin" / "llvm-objdump"
    return str(near if near.exists() else "/opt/rocm/llvm/bin/llvm-objdump")


def _scalars(operands: str) -> set[int]:
    found = {int(n) for n in re.findall(r"\bs(\d+)\b", operands)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", operands):
        found |= set(range(int(a), int(b) + 1))
    return found


def early_reads(listing: str) -> list[str]:
    """The memory instructions of a listing that come too early behind a vector write of a scalar that they read."""
    found, function = [], ""
    written: dict[int, int] = {}  # scalar register -> wait states since a vector instruction wrote it
    for line in listing.splitlines():
        label = re.match(r"(?:[0-9a-f]+ )?<(\w+)>:", line.strip())
        if label:
            function, written = label.group(1), {}
            continue
        text = line.split("//")[0].strip()
        if not text or not re.match(r"[a-z]+_\w+", text):
            continue
        op, _, operands = text.partition(" ")
        if op.startswith(MEMORY):
            for r in sorted(_scalars(operands) & {r for r, n in written.items() if n < NEEDED}):
                found.append(f"{function}: {text} (s{r} written {written[r]} wait states before)")
        passed = int(operands, 0) + 1 if op == "s_nop" else 1
        written = {r: n + passed for r, n in written.items() if n + passed < NEEDED}
        if op.startswith("v_"):
            written |= dict.fromkeys(_scalars(operands.split(",")[0]), 0)
        elif op.startswith("s_"):  # (a scalar instruction's result needs no wait)
            for r in _scalars(operands.split(",")[0]):
                written.pop(r, None)
    return found


def test_the_check_finds_early_reads():
    near = "<f>:\n v_readfirstlane_b32 s6, v1\n s_mov_b32 m0, s9\n s_nop {}\n buffer_load_dwordx4 v2, s[4:7], 0 offen lds\n"
    assert len(early_reads(near.format(0))) == 1 and len(early_reads(near.format(2))) == 1
    assert early_reads(near.format(3)) == []
    assert early_reads("<f>:\n v_readfirstlane_b32 s8, v1\n buffer_load_dword v2, v3, s[4:7], 0 offen\n") == []
    assert len(early_reads("<f>:\n v_readlane_b32 s8, v1, 3\n buffer_load_dword v2, v3, s[4:7], s8 offen\n")) == 1


def test_memory_instructions_wait_for_scalars_that_vector_instructions_wrote(tmp_path):
    lib = tmp_path / LIB.name
    shutil.copy(LIB, lib)
    subprocess.run([_objdump(), "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    images = sorted(p for p in tmp_path.iterdir() if p.name.endswith("gfx950"))
    assert images
    found, loads = [], 0
    for image in images:
        res = subprocess.run([_objdump(), "-d", "--no-show-raw-insn", str(image)], check=True, capture_output=True, text=True)
        loads += len(re.findall(r"\bbuffer_load_\w+ .*\blds\b", res.stdout))
        found += early_reads(res.stdout)
    assert loads > 100, loads  # (the listing is read: the kernels' loads straight into LDS are there)
    assert not found, f"{len(found)} early reads, the first: {found[:5]}"
