"""Wait states in the library's own kernels, read from the disassembly of the built libamdsplat.so.

A vector-memory instruction that reads a scalar register needs five wait states after a vector
instruction wrote it (v_readfirstlane and the like); the hardware does not wait by itself. The compiler
keeps to this among its own instructions, but does not look into inline assembly: a copy to LDS written
out there has to bring its wait along. Straight-line order is followed, which is how the compiler lays
out a resource and the copies that use it."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from amdsplat import _lib

TOOL = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")) if p and Path(p).exists()), None)
NEEDED = 5


def scalars(operand):
    """Numbers of the scalar registers that an operand names."""
    m = re.fullmatch(r"s(\d+)", operand)
    if m:
        return [int(m.group(1))]
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    return range(int(m.group(1)), int(m.group(2)) + 1) if m else []


def short_waits(lines):
    """(instruction, register, wait states since its vector write) of every read that comes too early."""
    age, found = {}, []  # scalar register -> wait states since a vector instruction wrote it
    for line in lines:
        line = line.split("//")[0].split(";")[0].strip()
        if not line or line.endswith(":"):
            continue
        name, _, rest = line.partition(" ")
        operands = re.findall(r"s\[\d+:\d+\]|\bs\d+\b|\bv\[\d+:\d+\]|\bv\d+\b|[^\s,]+", rest)
        if re.match(r"(buffer|global|flat|scratch|tbuffer)_", name):
            for o in operands:
                found += [(line, r, age[r]) for r in scalars(o) if age.get(r, NEEDED) < NEEDED]
        took = int(rest, 0) + 1 if name == "s_nop" else 1
        age = {r: n + took for r, n in age.items() if n + took < NEEDED}
        if name.startswith("v_"):
            # a vector instruction's scalar results: the first operand, or the carry behind the first
            wrote = operands[:1] + (operands[1:2] if re.search(r"_co_|div_scale", name) else [])
            for o in wrote:
                age.update((r, 0) for r in scalars(o))
        elif name.startswith("s_") and operands:
            for r in scalars(operands[0]):
                age.pop(r, None)
    return found


def test_short_waits_are_found():
    resource = ["v_readfirstlane_b32 s40, v1", "s_mov_b32 m0, s3"]
    load = "buffer_load_dwordx4 v2, s[40:43], 0 offen lds"
    assert [x[1:] for x in short_waits(resource + ["s_nop 0", load])] == [(40, 2)]
    assert [x[1:] for x in short_waits(resource + ["s_nop 2", load])] == [(40, 4)]
    assert short_waits(resource + ["s_nop 3", load]) == []
    assert short_waits(["v_readfirstlane_b32 s44, v1", load]) == []
    assert short_waits(["v_readfirstlane_b32 s40, v1", "s_mov_b32 s40, s7", load]) == []
    assert [x[1:] for x in short_waits(["v_cmp_lt_u32_e64 s[40:41], v1, v2", load])] == [(40, 0), (41, 0)]
    assert [x[1:] for x in short_waits(["v_add_co_u32_e64 v1, s[42:43], v1, v2", load])] == [(42, 0), (43, 0)]


def test_assembly_leaves_m0_to_the_compiler():
    """The compiler keeps LDS bases and indexes in M0 and may reuse what it put there: a block that needs a
    value in M0 takes it as an input and writes nothing to it."""
    blocks = []
    for path in sorted((Path(_lib.__file__).resolve().parent.parent / "csrc").iterdir()):
        blocks += re.findall(r"asm volatile\((.*?)\);", path.read_text(), re.S)
    copies = [b for b in blocks if re.search(r" lds\"", b)]
    assert len(copies) == 2 and all('"{m0}"(' in b for b in copies), copies
    assert not [b for b in blocks if re.search(r"\bm0\s*,", b)]


@pytest.mark.skipif(TOOL is None, reason="no llvm-objdump")
def test_kernels_wait_for_their_scalars(tmp_path):
    lib = tmp_path / "lib.so"
    shutil.copy(_lib.LIB_PATH, lib)
    subprocess.run([TOOL, "--offloading", lib.name], cwd=tmp_path, check=True, capture_output=True)
    objects = sorted(p for p in tmp_path.glob("lib.so.*gfx950") if p.stat().st_size)
    assert objects
    kernels, bad = 0, []
    for obj in objects:
        text = subprocess.run([TOOL, "-d", "--no-show-raw-insn", "--no-leading-addr", str(obj)], check=True,
                              capture_output=True, text=True).stdout
        name, body = None, []
        for line in [*text.splitlines(), "<end>:"]:
            m = re.match(r"(?:[0-9a-f]+ )?<([^>]+)>:$", line)
            if not m:
                body.append(line)
                continue
            if name:
                kernels += 1
                bad += [(name, *x) for x in short_waits(body)]
            name, body = m.group(1), []
    assert kernels > 100
    assert not bad, (len(bad), sorted({x[0] for x in bad})[:20], bad[:6])
