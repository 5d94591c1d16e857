"""Wait states of the LDS DMA loads that are written in inline asm, in the library as it was built.

The compiler's hazard recogniser does not look into inline asm, so two distances that the
ISA asks for are the source's own: a vector-memory load with an LDS destination reads M0
one wait state after a scalar instruction wrote it at the earliest, and a scalar register
that a vector instruction wrote (v_readfirstlane, or v_readlane where a descriptor was
spilled) five.  Read from the disassembly, over every path into each load.
"""
from __future__ import annotations

import os
import re
import shutil
import struct
import subprocess

import pytest

from h3attn import _lib

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The gfx950 code objects bundled in a shared library."""
    data = open(path, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        p = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            off, size, n = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + n] and size:
                yield data[at + off:at + off + size]
            p += 24 + n
        at = data.find(MAGIC, at + 24)


def instructions(elf, tmp):
    """(address, text) of a code object's instructions, branch targets as absolute addresses."""
    tmp.write_bytes(elf)
    out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(tmp)], capture_output=True, text=True, check=True)
    start, res = {}, []
    for line in out.stdout.splitlines():
        head = re.match(r"([0-9a-f]+) <(.*)>:$", line)
        if head:
            start[head[2]] = int(head[1], 16)
            continue
        text, _, note = line.partition("//")
        addr = re.match(r"\s*([0-9A-F]+):", note)
        if not addr:
            continue
        text = text.strip()
        if text.startswith(("s_branch", "s_cbranch")):
            to = re.search(r"<(.*?)(?:\+0x([0-9a-f]+))?>\s*$", note)
            text += f" -> {start[to[1]] + int(to[2] or '0', 16)}"
        res.append((int(addr[1], 16), text))
    return res


def registers(text):
    """Scalar registers among an instruction's operands."""
    regs = {int(n) for n in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        regs.update(range(int(a), int(b) + 1))
    return regs


def scalars_written(text):
    """Scalar registers that a vector instruction writes: its first operand, or a carry or the like after it."""
    two = re.match(r"v_\w+_co_|v_div_scale|v_mad_[iu]64", text)
    return registers(",".join(text.split(",")[:2 if two else 1]))


def broken(code):
    """LDS DMA loads of a code object, and those of them that come too early."""
    into = {}
    for i, (_, text) in enumerate(code):
        if " -> " in text:
            into.setdefault(int(text.split(" -> ")[1]), []).append(i)

    def too_early(i, regs):
        """Whether some path into instruction i writes what it reads within the distance."""
        todo, seen = [(i, 0)], set()
        while todo:
            j, waited = todo.pop()
            before = list(into.get(code[j][0], []))
            if j > 0 and not code[j - 1][1].startswith(("s_branch", "s_endpgm", "s_setpc")):
                before.append(j - 1)
            for b in before:
                text = code[b][1]
                if re.match(r"s_\w+ m0\b", text) and waited < 1:
                    return text
                if text.startswith("v_") and waited < 5 and scalars_written(text) & regs:
                    return text
                nop = re.match(r"s_nop (\d+)", text)
                w = waited + (int(nop[1]) + 1 if nop else 1)
                if w < 5 and (b, w) not in seen:
                    seen.add((b, w))
                    todo.append((b, w))
        return None

    loads = [i for i, (_, t) in enumerate(code) if re.match(r"(buffer_load.*\blds\b|global_load_lds)", t)]
    bad = []
    for i in loads:
        text = code[i][1]
        why = too_early(i, registers(text) if text.startswith("buffer") else set())
        if why:
            bad.append(f"{code[i][0]:#x}: {text} after {why}")
    return loads, bad


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="llvm-objdump is not installed")
@pytest.mark.parametrize("path", [_lib.LIB_PATH, _lib.PROF_LIB_PATH], ids=os.path.basename)
def test_lds_dma_loads_wait(path, tmp_path):
    if path == _lib.PROF_LIB_PATH and not os.path.exists(path):
        pytest.skip("the phase-profile library is not built")
    total, bad = 0, []
    for n, elf in enumerate(code_objects(path)):
        loads, early = broken(instructions(elf, tmp_path / f"{n}.elf"))
        total += len(loads)
        bad += early
    assert total > 100  # they are found at all
    assert not bad, f"{len(bad)} of {total} loads: " + "; ".join(bad[:5])


def test_paths_are_followed():
    """The search itself: straight on, across a branch, and with waits in between."""
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    run = lambda *texts: len(broken([(4 * i, t) for i, t in enumerate(texts)])[1])  # noqa: E731
    assert run("s_mov_b32 m0, s1", load) == 1
    assert run("s_mov_b32 m0, s1", "s_nop 0", load) == 0
    assert run("v_readfirstlane_b32 s6, v3", "s_nop 3", load) == 1
    assert run("v_readfirstlane_b32 s6, v3", "s_nop 4", load) == 0
    assert run("v_readfirstlane_b32 s9, v3", "s_nop 0", load) == 0
    assert run("v_readlane_b32 s4, v3, 5", "s_branch 9 -> 16", "s_nop 7", "s_nop 7", "s_nop 1", load) == 1
    assert run("v_readlane_b32 s4, v3, 5", "s_branch 9 -> 16", "s_nop 7", "s_nop 7", "s_nop 3", load) == 0
    assert run("v_add_co_u32_e64 v1, s[4:5], v2, v3", "s_nop 3", load) == 1
    assert run("v_cmp_lt_u32_e64 s[6:7], v2, v3", "s_nop 4", load) == 0
