"""Inline assembly next to matrix and cross-lane instructions.

The compiler keeps the waits that the hardware asks for between the instructions it
knows, and takes no part in this for instructions written as text: such a one may
read a register before the matrix instruction ahead of it has written it, and a
cross-lane read (DPP, permlane) may come before such a one's result. So the built
code is searched: no text instruction of the vector unit reads a matrix result, or
writes what a cross-lane instruction reads, fewer issue slots away than any such
wait is long."""
import re
import subprocess

import pytest

from muserve_amd import build

MATRIX_SLOTS = 20  # the longest wait of a 16-pass matrix instruction is 18 slots
LANES_SLOTS = 3    # of a cross-lane read, 2

SOURCES = [p for p in sorted(build.CSRC.glob("*.hip")) if "mfma" in p.read_text()]


def registers(operand):
    operand = operand.strip().strip("-|")
    m = re.fullmatch(r"v\[(\d+):(\d+)\]", operand)
    if m:
        return range(int(m[1]), int(m[2]) + 1)
    m = re.fullmatch(r"v(\d+)", operand)
    return [int(m[1])] if m else []


def findings(text):
    """(function, instruction, writer) of every read that comes too early."""
    bad, function, slot, inside = [], None, 0, False
    matrix, written = {}, {}  # register: (slot, instruction)
    for line in text.splitlines():
        line = line.strip()
        label = re.match(r"^(_Z\w+):", line)
        if label:
            function, slot, matrix, written = label[1], 0, {}, {}
        if "ASMSTART" in line:
            inside = True
        elif "ASMEND" in line:
            inside = False
        line = line.split(";")[0].strip()
        if not line or line.startswith(".") or line.endswith(":"):
            continue
        name, _, rest = line.partition(" ")
        slot += int(rest, 0) + 1 if name == "s_nop" else 1
        if not name.startswith(("v_", "ds_", "global_", "buffer_", "scratch_")):
            continue
        operands = re.split(r",\s*|\s+(?=quad_perm|row_|bank_mask|op_sel)", rest)
        lanes = "row_" in rest or "quad_perm" in rest or name.startswith("v_permlane")
        reads = operands[0 if name.startswith("v_permlane") else 1:]
        for r in sorted({r for o in reads for r in registers(o)}):
            if inside and name.startswith("v_") and r in matrix \
                    and slot - matrix[r][0] < MATRIX_SLOTS:
                bad.append((function, line, matrix[r][1]))
            if lanes and r in written and slot - written[r][0] < LANES_SLOTS:
                bad.append((function, line, written[r][1]))
        for r in registers(operands[0]):
            matrix.pop(r, None)
            written.pop(r, None)
            if name.startswith("v_mfma"):
                matrix[r] = (slot, line)
            elif inside and name.startswith("v_"):
                written[r] = (slot, line)
    return bad


def test_the_search_finds_what_it_is_for():
    early = """
_Zkernel:
  v_mfma_f32_16x16x4_f32 v[4:7], v1, v2, v[8:11]
  ;;#ASMSTART
  v_max3_f32 v12, v12, |v4|, |v5|
  ;;#ASMEND
  s_nop 0
  v_max_f32_dpp v3, v12, v12 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf
"""
    assert len(findings(early)) == 3  # (two registers of the matrix result)
    late = early.replace("  ;;#ASMSTART", "  s_nop 15\n  s_nop 3\n  ;;#ASMSTART")
    assert len(findings(late)) == 1
    assert not findings(late.replace("s_nop 0", "s_nop 1"))
    assert not findings(early.replace(";;#ASMSTART", "").replace(";;#ASMEND", ""))


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.stem)
def test_text_instructions_keep_their_distance(source, tmp_path):
    out = tmp_path / "code.s"
    flags = [*build.HIP_FLAGS, *build.EXTRA_FLAGS.get(source.stem, [])]
    subprocess.run([build.hipcc(), *flags, "--offload-device-only", "-S", str(source), "-o", str(out)],
                   check=True, capture_output=True)
    text = out.read_text()
    assert "v_mfma" in text
    assert not findings(text)
