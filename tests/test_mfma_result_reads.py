"""No instruction of the built kernels touches what an MFMA leaves in registers before it is there.

Between such a product and a vector instruction that reads or writes its result, a memory or LDS instruction that reads it, or a product that takes it as A or B, the hardware needs
wait states: 8 behind 16x16x32 (four passes), 12 behind 32x32x16 (eight).  The compiler counts them, but has left them out along a branch that skips what stood in
between.  (A product that takes a result as C waits by itself.)"""
import os
import re
import shutil
import subprocess

import pytest

from easyllm_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
NEEDED = {"v_mfma_f32_16x16x32": 8, "v_mfma_f32_32x32x16": 12}
PRODUCT = re.compile(r"v_s?mfma\S*?_(\d+x\d+x\d+)|v_smfmac")
MEMORY = re.compile(r"(buffer|global|flat|scratch|ds|image|tbuffer)_")
ONLY_WRITES_FIRST = re.compile(r"(buffer|global|flat|scratch)_load_|ds_(read|bpermute|permute|swizzle|consume|append)")
REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(operands):
    return {(kind, i) for kind, first, last, one in REG.findall(operands) for i in range(int(first or one), int(last or one) + 1)}


def touched(op, operands):
    """The registers that an instruction must not meet a product's unfinished result in."""
    if PRODUCT.match(op):
        return registers(",".join(operands.split(",")[1:3]))
    if op.startswith("v_"):
        return registers(operands)  # (the first is written, by some, as v_permlane16_swap or v_fmac, read too; neither may come early)
    if MEMORY.match(op):
        first, _, rest = operands.partition(",")
        return registers(rest if ONLY_WRITES_FIRST.match(op) and " lds" not in operands else operands)
    return set()


def needed(text):
    return next((n for shape, n in NEEDED.items() if text.startswith(shape)), 0)


def early(code):
    """code: (address, instruction, address it branches to or None), in order -> (product, instruction) pairs that are too close"""
    at = {a: i for i, (a, _, _) in enumerate(code)}
    split = [text.partition(" ")[::2] for _, text, _ in code]
    uses = [touched(op, operands) for op, operands in split]
    hits = []
    for i, (op, operands) in enumerate(split):
        states = needed(op)
        if not states:
            continue
        result = registers(operands.split(",")[0])
        todo, seen = [(i + 1, 0)], set()
        while todo:
            j, waited = todo.pop()
            while j < len(code) and waited < states and (j, waited) not in seen:
                seen.add((j, waited))
                here, args = split[j]
                if here == "s_endpgm":
                    break
                if uses[j] & result:
                    hits.append((code[i][1], code[j][1]))
                    break
                if code[j][2] in at:
                    todo.append((at[code[j][2]], waited + 1))
                    if here == "s_branch":
                        break
                waited += int(args) + 1 if here == "s_nop" else 1
                j += 1
    return hits


SMALL, LARGE = "v_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], 0", "v_mfma_f32_32x32x16_bf16 a[0:15], v[8:11], v[12:15], a[0:15]"


@pytest.mark.parametrize("reader", [
    "v_add_f32_e32 v1, v2, v5", "v_permlane16_swap_b32_e32 v4, v20", "v_permlane32_swap_b32_e32 v20, v7", "v_swap_b32 v5, v30", "v_fmac_f32_e32 v5, v1, v2",
    "v_dot2c_f32_bf16_e32 v6, v1, v2", "v_mov_b32_e32 v7, v1", "v_readfirstlane_b32 s3, v6", "v_cmp_gt_f32_e32 vcc, v4, v1", "v_mfma_f32_16x16x32_bf16 v[20:23], v[4:7], v[12:15], 0",
    "v_mfma_f32_32x32x16_bf16 a[0:15], v[8:11], v[6:9], a[0:15]", "flat_store_dword v[0:1], v5", "global_store_dwordx4 v0, v[4:7], s[0:1]", "global_atomic_add v0, v4, s[0:1]",
    "buffer_store_dwordx4 v[4:7], v0, s[0:3], 0 offen", "buffer_load_dwordx4 v5, s[0:3], 0 offen lds", "buffer_load_dword v1, v5, s[0:3], 0 offen", "ds_bpermute_b32 v1, v2, v5",
    "ds_write_b128 v1, v[4:7]", "ds_read_b128 v[20:23], v4", "ds_add_u32 v1, v5", "scratch_store_dword off, v6, s0"])
def test_the_scan_finds_what_it_looks_for(reader):
    assert early([(0, SMALL, None), (8, reader, None)])
    assert early([(0, SMALL, None), (8, "s_nop 6", None), (12, reader, None)])
    assert not early([(0, SMALL, None), (8, "s_nop 7", None), (12, reader, None)])
    jump = [(0, SMALL, None), (8, "s_cbranch_vccnz 9", 24), (12, "s_nop 15", None), (16, "s_nop 15", None), (24, reader, None)]
    assert early(jump) and not early(jump[:1] + jump[2:])


def test_the_scan_lets_pass_what_waits_by_itself():
    assert not early([(0, SMALL, None), (8, "v_mfma_f32_16x16x32_bf16 v[4:7], v[20:23], v[12:15], v[4:7]", None)])
    assert not early([(0, SMALL, None), (8, "v_add_f32_e32 v1, v2, v3", None), (12, "ds_read_b128 v[20:23], v30", None), (16, "s_endpgm", None), (20, "v_mov_b32_e32 v4, v1", None)])
    read = "v_accvgpr_read_b32 v1, a9"
    assert early([(0, LARGE, None), (8, "s_nop 10", None), (12, read, None)]) and not early([(0, LARGE, None), (8, "s_nop 11", None), (12, read, None)])


def test_results_are_not_touched_early(tmp_path):
    if not os.path.exists(OBJDUMP) or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("needs the built library and the ROCm disassembler")
    subprocess.run([OBJDUMP, "--offloading", shutil.copy(_lib.LIB_PATH, tmp_path)], cwd=tmp_path, check=True, capture_output=True)
    products, hits = {shape: 0 for shape in NEEDED}, []
    for f in os.listdir(tmp_path):
        if "gfx950" not in f:
            continue
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        base, kernel, code = {}, None, []
        for line in out.splitlines() + ["0 <end>:"]:
            label = re.match(r"([0-9a-f]+) <(.*)>:", line)
            if label:
                if any(PRODUCT.match(t) for _, t, _ in code):
                    hits += [(kernel,) + h for h in early(code)]
                kernel, code = label.group(2), []
                base[kernel] = int(label.group(1), 16)
                continue
            m = re.match(r"\t(.*?)\s*// ([0-9A-F]+):(?:\s+[0-9A-F]{8})*(?:\s*<(.+?)(?:\+0x([0-9a-f]+))?>)?", line)
            if m:
                target = base[m.group(3)] + int(m.group(4) or "0", 16) if m.group(3) in base else None
                code.append((int(m.group(2), 16), m.group(1), target))
                if PRODUCT.match(m.group(1)):
                    shape = next((s for s in NEEDED if m.group(1).startswith(s)), None)
                    assert shape, "a product of another shape: " + m.group(1)
                    products[shape] += 1
    assert all(products.values()), products
    assert not hits, (len(hits), hits[:5])
