"""The machine code of the vocabulary kernels, as built: what the compiler does not
look after because it is written as assembler (``ace_mma.hpp``).

gfx950 does not hold back a vector memory instruction for scalar registers that a
vector instruction writes (``v_readfirstlane``): five wait states must lie between
the two, or the address may be the old one.  The compiler keeps them for its own
instructions, and sees nothing of those inside an ``asm`` block."""

from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path
from typing import Dict, Iterator, List, Set, Tuple

import pytest

from ace_kernels import _lib

WAIT = 5  # wait states from a vector write of a scalar register to a vector memory read of it
OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")) if p and Path(p).exists()), None)
_LINE = re.compile(r"^\t(\S+)(?: (.*?))?\s*// ([0-9A-F]+): ")
_LABEL = re.compile(r"^([0-9a-f]{16}) <(.+)>:$")
_TARGET = re.compile(r"<.+\+0x([0-9a-f]+)>$|<([^+>]+)>$")


def _code_objects(path: Path) -> Iterator[bytes]:
    """The gfx950 code objects of the built library."""
    data = path.read_bytes()
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", 0
    while (at := data.find(magic, at)) >= 0:
        pos = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            off, size, length = struct.unpack_from("<QQQ", data, pos)
            target = data[pos + 24:pos + 24 + length]
            pos += 24 + length
            if b"gfx950" in target and size:
                yield data[at + off:at + off + size]
        at += len(magic)


Function = List[Tuple[int, str, str]]  # address, mnemonic, operands


def _functions(text: str) -> Dict[str, Tuple[int, Function]]:
    out: Dict[str, Tuple[int, Function]] = {}
    here: Function = []
    for line in text.splitlines():
        if m := _LABEL.match(line):
            here = []
            out[m[2]] = (int(m[1], 16), here)
        elif m := _LINE.match(line):
            # a branch's target is in the comment behind the encoding
            tail = line[line.index("//"):]
            here.append((int(m[3], 16), m[1], (m[2] or "") + (" " + tail if m[1].startswith("s_") and "branch" in m[1] else "")))
    return out


def _scalars(operand: str) -> Set[int]:
    """The scalar registers that an operand names; vcc as 1000 and 1001."""
    if m := re.fullmatch(r"s\[(\d+):(\d+)\]", operand):
        return set(range(int(m[1]), int(m[2]) + 1))
    if m := re.fullmatch(r"s(\d+)", operand):
        return {int(m[1])}
    return {"vcc": {1000, 1001}, "vcc_lo": {1000}, "vcc_hi": {1001}}.get(operand, set())


def _operands(text: str) -> List[str]:
    return [o for part in re.split(r",\s*", text.split("//")[0].strip()) for o in part.split()[:1]]


def hazards(start: int, code: Function) -> List[str]:
    """Vector memory instructions that may read a scalar register fewer than
    ``WAIT`` wait states after a vector instruction wrote it, along any path."""
    index = {a: i for i, (a, _, _) in enumerate(code)}
    before: Dict[int, List[int]] = {i: [] for i in range(len(code))}
    for i, (_, op, args) in enumerate(code):
        if op not in ("s_branch", "s_endpgm", "s_setpc_b64") and i + 1 < len(code):
            before[i + 1].append(i)
        if "branch" in op and (m := _TARGET.search(args)):
            to = index.get(start + int(m[1], 16) if m[1] else start)
            assert to is not None, args
            before[to].append(i)
    found = []
    for i, (_, op, args) in enumerate(code):
        if not op.startswith(("global_", "buffer_", "scratch_", "flat_")):
            continue
        reads = set().union(set(), *(_scalars(o) for o in _operands(args)))
        todo = [(p, 0, reads) for p in before[i]] if reads else []
        seen: Set[Tuple[int, int]] = set()
        while todo:
            at, states, left = todo.pop()
            if states >= WAIT or (at, states) in seen:
                continue
            seen.add((at, states))
            _, op2, args2 = code[at]
            out = _operands(args2)
            # most vector instructions write their first operand, those with a carry two
            writes = set().union(set(), *(_scalars(o) for o in out[:2 if "_co_" in op2 else 1]))
            if op2.startswith("v_") and writes & left:
                found.append(f"{code[i][1]} {args.strip()}: {states} wait states after {op2} {args2.strip()}")
            if op2.startswith("s_") and not op2.startswith(("s_cmp", "s_bitcmp", "s_waitcnt", "s_nop", "s_barrier")):
                left = left - writes  # a scalar instruction's result is waited for
            states += int(args2.split()[0], 0) + 1 if op2 == "s_nop" else 1
            todo += [(p, states, left) for p in before[at]]
    return found


def test_the_search_itself() -> None:
    def at(*lines: str) -> Function:
        return [(4 * i, line.split(" ", 1)[0], line.split(" ", 1)[1] if " " in line else "") for i, line in enumerate(lines)]

    load = "global_load_lds_dwordx4 v1, s[40:41]"
    near = at("v_readfirstlane_b32 s41, v2", "s_mov_b32 m0, s9", "s_nop 0", load)
    assert len(hazards(0, near)) == 1 and "2 wait states" in hazards(0, near)[0]
    assert not hazards(0, at("v_readfirstlane_b32 s41, v2", "s_mov_b32 m0, s9", "s_nop 3", load))
    assert hazards(0, at("v_readfirstlane_b32 s41, v2", "s_mov_b32 m0, s9", "s_nop 2", load))
    assert not hazards(0, at("v_readfirstlane_b32 s42, v2", load))
    assert not hazards(0, at("v_readfirstlane_b32 s41, v2", "s_add_u32 s41, s3, s4", "s_mov_b32 s40, s2", load))
    assert hazards(0, at("v_cmp_gt_u32_e64 s[40:41], s2, v3", load))
    # through a branch: the load follows the write at the loop's end
    loop = at(load, "v_mov_b32_e32 v1, v2", "v_readfirstlane_b32 s40, v2", "s_cbranch_scc1 0 // 0000000C: BF85FFFC <k>", "s_endpgm")
    assert len(hazards(0, loop)) == 1


def test_addresses_in_scalar_registers_have_settled(tmp_path) -> None:
    if OBJDUMP is None:
        pytest.skip("no llvm-objdump")
    kernels = loads = 0
    wrong = []
    for n, elf in enumerate(_code_objects(_lib.LIB_PATH)):
        if b"grad_kernel" not in elf:
            continue
        path = tmp_path / f"{n}.co"
        path.write_bytes(elf)
        text = subprocess.run([OBJDUMP, "-d", str(path)], check=True, capture_output=True, text=True).stdout
        for name, (start, code) in _functions(text).items():
            kernels += "grad_kernel" in name
            loads += sum(op.startswith("global_load_lds") for _, op, _ in code)
            wrong += [f"{name}: {h}" for h in hazards(start, code)]
    assert kernels >= 3 and loads  # the three element types
    assert not wrong, f"{len(wrong)}, the first: " + "\n".join(wrong[:5])
