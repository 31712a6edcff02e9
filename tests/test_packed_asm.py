"""CPU only: what the pipelined kernel for packed prompts needs of the generated gfx950 code and the compiler does not
promise (its matrix instructions are issued from inline asm, see tests/test_kernel_asm.py)."""
import importlib.util
import os
import re

import pytest

from conftest import ROOT


def _load(name, *path):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, *path))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def kernels():
    path = _load("fa_build", "flash-attention_amd", "build.py").build_device_asm(unit="flash_packed")
    text = open(path).read()
    # the compiler pads the matrix instructions it issues itself (the path that takes rows by themselves): only those
    # between its ASMSTART and ASMEND marks are inline asm
    inside, lines = False, []
    for line in text.split("\n"):
        s = line.strip()
        inside = True if s.startswith(";;#ASMSTART") else False if s.startswith(";;#ASMEND") else inside
        lines.append(line if inside else line.replace("v_mfma_", "v_padded_mfma_"))
    text = "\n".join(lines)
    hazards = _load("mfma_hazards", "tools", "mfma_hazards.py")
    found = {n: l for n, l in hazards.kernels(text).items() if "attn_fwd_kernel_packed" in n}
    assert len(found) == 24, list(found)      # two layouts and the cut items of one, two head-dim tiles, two types, causal or not
    return text, hazards, found


def test_no_spills_to_memory(kernels):
    text, _, _ = kernels
    assert all(v == "0" for v in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text))
    assert not re.search(r"\.private_segment_fixed_size:\s+[1-9]", text)


def test_matrix_instruction_hazards(kernels):
    """Operands written just before, results read too early, scalar operands a vector instruction just wrote."""
    _, hazards, found = kernels
    for name, lines in found.items():
        assert not hazards.result_hazards(lines), name
        assert not hazards.hazards(lines, window=3), name
        assert not hazards.scalar_operand_hazards(lines), name


def test_accumulators_stay_in_place(kernels):
    """O^T, Q and the row sums never move between the register files in the steps of the tile iterations: no block with
    more matrix instructions than the prologue and the last product (whose instructions are padded) holds a move from or to
    a register of a matrix instruction.  (The kernels that cut items park a value or two in others.)"""
    _, _, found = kernels

    def registers(operand):
        m = re.fullmatch(r"a\[(\d+):(\d+)\]|a(\d+)", operand.strip())
        return set() if not m else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))

    for name, lines in found.items():
        padded = (32 if "Li128E" in name else 16) // (2 if "4m16h" in name else 1)
        blocks, cur = [], []
        for l in lines:
            if l.startswith(".LBB"):
                blocks.append(cur)
                cur = []
            cur.append(l)
        blocks.append(cur)
        steps = [b for b in blocks if sum("v_mfma_f32_16x16x32" in l for l in b) > padded]
        assert len(steps) >= 6, (name, len(steps))
        held = {r for b in steps for l in b if l.startswith("v_mfma_") for x in l.split(None, 1)[1].split(",") for r in registers(x)}
        assert held, name
        for b in steps:
            for l in b:
                if l.startswith("v_accvgpr_"):
                    moved = {r for x in l.split(None, 1)[1].split(",") for r in registers(x)}
                    assert not moved & held, (name, l)
                    assert "Lb1EEEv" in name, (name, l)
