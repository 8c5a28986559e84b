"""Inline assembly beside matrix instructions: the compiler counts wait states for the instructions that it emits itself and
none for those inside an asm block, but it may give a block's outputs registers that a matrix instruction just issued still
writes or reads as its C operand. So a block waits before its first write: 8 states behind the f16 products for their
result (written or read), 3 for their C operand. Read off the assembly that the compiler makes of the sources here."""
from __future__ import annotations

import re
import subprocess

import pytest

from glint_amd import build

RESULT, C_OPERAND = 8, 3  # wait states of a 4-pass matrix instruction on gfx950


def regs(operand):
    """Vector registers of an operand: v7, -v7, |v7|, v[4:7], a[0:3]."""
    m = re.search(r"([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.search(r"(?<![a-z0-9_])([va])(\d+)\b", operand)
    return {m[1] + m[2]} if m else set()


def states(line):
    m = re.match(r"s_nop (\d+)", line)
    return int(m[1]) + 1 if m else 1


def short_waits(asm):
    """(kernel, line, instruction, states kept, states needed) of instructions in asm blocks that come too soon behind a
    matrix instruction of f16 operands, and how many vector instructions in such blocks were looked at."""
    found, looked = [], 0
    kernel, inside, ahead = "", False, []  # ahead: (states since, result, C operand) of the last matrix instructions
    for at, line in enumerate(asm.split("\n"), 1):
        m = re.match(r"(_Z\w+):", line)
        if m:
            kernel, ahead = m[1], []
        if "#ASMSTART" in line or "#ASMEND" in line:
            inside = "#ASMSTART" in line
            continue
        line = line.split(";")[0].strip()
        if not line or line[0] == "." or line.endswith(":"):
            continue
        op, _, rest = line.partition(" ")
        # operands, with the brackets of a range kept whole
        args = [a.strip() for a in rest.split(",")]
        if inside and op.startswith("v_"):
            looked += 1
            writes, reads = regs(args[0]), set().union(*map(regs, args[1:]), set())
            for since, result, c in ahead:
                need = RESULT if (writes | reads) & result else (C_OPERAND if writes & c else 0)
                if since < need:
                    found.append((kernel, at, line, since, need))
        n = states(line)
        ahead = [(s + n, r, c) for s, r, c in ahead if s + n < RESULT]
        if op in ("v_mfma_f32_16x16x32_f16", "v_mfma_f32_16x16x16_f16"):
            ahead.append((0, regs(args[0]), regs(args[3])))
    return found, looked


def test_reads_assembly():
    mfma = "_Zk:\n\tv_mfma_f32_16x16x32_f16 v[4:7], v[0:3], v[8:11], v[12:15]\n"
    block = "\t;;#ASMSTART\n\ts_nop {}\n\tv_fma_mixlo_f16 {}, v20, {}, 0\n\t;;#ASMEND\n"
    for nop, out, arg, kept in ((1, "v5", "v21", 2), (6, "v5", "v21", 7), (7, "v5", "v21", None), (1, "v12", "v21", 2),
                                (2, "v12", "v21", None), (0, "v16", "v21", None), (0, "v0", "v21", None), (3, "v16", "-v4", 4)):
        found, looked = short_waits(mfma + block.format(nop, out, arg))
        assert looked == 1 and [f[3] for f in found] == ([] if kept is None else [kept])


@pytest.mark.parametrize("source", ["gla_decode_q8.hip", "gla_q4.hip"])
def test_asm_blocks_wait_for_matrix_instructions(source, tmp_path):
    out = tmp_path / "k.s"
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / source), "-o", str(out)],
                   check=True, capture_output=True)
    found, looked = short_waits(out.read_text())
    assert looked > 0
    assert not found, found[:5]
