"""The built kernels read what a 16x16x32 MFMA leaves in registers no sooner than eight wait states behind it.

The hardware needs them between such a product and a vector instruction or a store that reads its result; the compiler counts them, but has left them out along a
branch that skips what stood in between (a product of few rows came out with wrong last elements)."""
import os
import re
import shutil
import subprocess

import pytest

from easyllm_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
NEEDED = 8
REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(operands):
    out = set()
    for kind, first, last, one in REG.findall(operands):
        out |= {(kind, i) for i in range(int(first or one), int(last or one) + 1)}
    return out


def early_reads(code):
    """code: (address, instruction, address it branches to or None), in order -> (product, reader) pairs that are too close"""
    at = {a: i for i, (a, _, _) in enumerate(code)}
    hits = []
    for i, (_, text, _) in enumerate(code):
        if not text.startswith("v_mfma_f32_16x16x32"):
            continue
        result = registers(text.split(None, 1)[1].split(",")[0])
        todo, seen = [(i + 1, 0)], set()
        while todo:
            j, waited = todo.pop()
            while j < len(code) and waited < NEEDED and (j, waited) not in seen:
                seen.add((j, waited))
                _, here, target = code[j]
                op, _, operands = here.partition(" ")
                if op == "s_endpgm":
                    break
                if op.startswith("v_") and not op.startswith("v_mfma") and registers(operands.partition(",")[2]) & result:
                    hits.append((text, here))
                    break
                if re.match(r"(buffer_store|global_store|scratch_store|ds_write)", op) and registers(operands) & result:
                    hits.append((text, here))
                    break
                if target in at:
                    todo.append((at[target], waited + 1))
                    if op == "s_branch":
                        break
                waited += int(operands) + 1 if op == "s_nop" else 1
                j += 1
    return hits


def test_the_scan_finds_what_it_looks_for():
    mfma = (0, "v_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], 0", None)
    add = "v_add_f32_e32 v1, v2, v5"
    assert early_reads([mfma, (8, add, None)])
    assert not early_reads([mfma, (8, "s_nop 7", None), (16, add, None)])
    assert not early_reads([mfma, (8, "v_add_f32_e32 v5, v2, v1", None)])
    jump = [mfma, (8, "s_cbranch_vccnz 9", 24), (12, "s_nop 15", None), (16, "s_nop 15", None), (24, add, None)]
    assert early_reads(jump) and not early_reads(jump[:1] + jump[2:])


def test_results_are_not_read_early(tmp_path):
    if not os.path.exists(OBJDUMP) or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("needs the built library and the ROCm disassembler")
    subprocess.run([OBJDUMP, "--offloading", shutil.copy(_lib.LIB_PATH, tmp_path)], cwd=tmp_path, check=True, capture_output=True)
    products, hits = 0, []
    for f in os.listdir(tmp_path):
        if "gfx950" not in f:
            continue
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        base, kernel, code = {}, None, []
        for line in out.splitlines() + ["0 <end>:"]:
            label = re.match(r"([0-9a-f]+) <(.*)>:", line)
            if label:
                if any(t.startswith("v_mfma_f32_16x16x32") for _, t, _ in code):
                    products += 1
                    hits += [(kernel,) + h for h in early_reads(code)]
                kernel, code = label.group(2), []
                base[kernel] = int(label.group(1), 16)
                continue
            m = re.match(r"\t(.*?)\s*// ([0-9A-F]+):(?:\s+[0-9A-F]{8})*(?:\s*<(.+?)(?:\+0x([0-9a-f]+))?>)?", line)
            if m:
                target = base[m.group(3)] + int(m.group(4) or "0", 16) if m.group(3) in base else None
                code.append((int(m.group(2), 16), m.group(1), target))
    assert products >= 60, products
    assert not hits, hits[:5]
