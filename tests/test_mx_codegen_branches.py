"""The generated code of every MXFP4 product along its branches, both ways: no result of a matrix instruction is touched while it
is being written, and no matrix instruction reads an operand that a vector instruction has only just written."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocm_dev_amd", "csrc")
# Wait states (an instruction is one) from a 16 x 16 x 128 matrix instruction to a read of its result: four passes where both operands are
# E2M1, eight where one is E4M3; an overwrite by a vector instruction may come one earlier.  A vector instruction's result is
# an operand two later.
READ = {True: 8, False: 12}
OPERAND = 2


def _registers(text):
    regs = set()
    for kind, lo, hi, one in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        regs.update((kind, r) for r in (range(int(lo), int(hi) + 1) if lo else (int(one),)))
    return frozenset(regs)


def _functions(text):
    """{kernel: (instructions, {label: index})}"""
    out = {}
    for m in re.finditer(r"^(_ZN2sg\w+):[^\n]*\n(.*?)^\s*\.section", text, re.S | re.M):
        code, labels = [], {}
        for line in m.group(2).splitlines():
            line = line.split(";")[0].strip()
            if line.endswith(":"):
                labels[line[:-1]] = len(code)
            elif line and not line.startswith("."):
                code.append(line)
        out[m.group(1)] = code, labels
    return out


class Instruction:
    def __init__(self, text):
        self.text = text
        self.op, _, self.operands = text.replace("\t", " ").partition(" ")
        first, _, rest = self.operands.partition(",")
        self.matrix = self.op.startswith("v_mfma")
        self.vector = self.op.startswith("v_") and not self.matrix
        loads = "load" in self.op and "lds" not in self.op or self.op.startswith("ds_read")
        writes = self.matrix or loads or self.vector and not self.op.startswith(("v_cmp", "v_readlane", "v_readfirstlane"))
        written = _registers(first) if writes else frozenset()
        self.writes, self.reads = written, _registers(rest if written else self.operands)
        if self.op.startswith("v_swap"):
            self.writes = self.reads = _registers(self.operands)
        if self.matrix:
            # D, A, B, C, two scales
            parts = [_registers(p) for p in self.operands.split(" op_sel")[0].split(",")]
            self.sum, self.reads = parts[3], parts[1] | parts[2] | parts[4] | parts[5]
            self.fp4 = "blgp:4" in text
        self.states = int(self.operands) + 1 if self.op == "s_nop" else 1


def _walk(code, labels, start, limit, live, step):
    """step(instruction, live, states) -> (fault, live) for what can follow code[start] within `limit` wait states"""
    paths, seen, faults = [(start + 1, 0, live)], {}, []
    while paths:
        at, states, live = paths.pop()
        while at < len(code) and states < limit and live and seen.get((at, live), limit) > states:
            seen[at, live] = states
            i = code[at]
            if i.op.startswith(("s_endpgm", "s_setpc")):
                break
            fault, live = step(i, live, states)
            if fault:
                faults.append((code[start].text, i.text, states))
                break
            if i.op.startswith("s_cbranch"):
                paths.append((labels[i.operands], states + 1, live))
            states += i.states
            at = labels[i.operands] if i.op == "s_branch" else at + 1
    return faults


def early(code, labels):
    """(matrix instructions, accesses to their results and operands of theirs that come too early)"""
    code = [Instruction(t) for t in code]
    faults, matrix = [], 0
    for at, i in enumerate(code):
        if i.matrix:
            matrix += 1

            def touched(j, live, states):
                # a matrix instruction may overwrite a result, or take the very registers as its sum; any other use has to wait
                if j.matrix:
                    hit = j.reads & live or (j.sum & live and j.sum != i.writes)
                else:
                    hit = j.reads & live or (states < READ[i.fp4] - 1 and j.writes & live)
                return hit, live - j.writes
            faults += _walk(code, labels, at, READ[i.fp4], i.writes, touched)
        elif i.vector and i.writes:
            def used(j, live, states):
                return j.matrix and (j.reads | j.sum) & live, live - j.writes
            faults += _walk(code, labels, at, OPERAND, i.writes, used)
    return matrix, faults


def test_no_product_meets_another_instruction_too_early_along_any_branch():
    if not shutil.which("hipcc") and not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("no hipcc")
    subprocess.run(["make", "-s", "-C", CSRC, "obj/sg_mx_gemm.s"], check=True, capture_output=True)
    kernels = _functions(open(os.path.join(CSRC, "obj", "sg_mx_gemm.s")).read())
    counted = {}
    for name, (code, labels) in kernels.items():
        matrix, faults = early(code, labels)
        assert not faults, "%s: %s is %d wait states in front of %s" % (name, faults[0][0], faults[0][2], faults[0][1])
        family = re.match(r"_ZN2sg\d+mx_(\w+?)_kernel", name).group(1)
        counted.setdefault(family, []).append(matrix)
    # both activation formats of every build; the kernel that adds a K split's sums multiplies nothing
    assert len(counted["gemm"]) == 12 and len(counted["tile"]) == 14 and len(counted["wide"]) == 12
    assert all(n > 0 for family in ("gemm", "tile", "wide") for n in counted[family]) and counted["sum"] == [0]


FP8 = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[10:13], v[20:27], a[0:3], v40, v41 op_sel:[1,0,0] op_sel_hi:[0,0,0] cbsz:4"
FP4 = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[10:13], v[20:23], a[0:3], v40, v41 op_sel_hi:[0,0,0] cbsz:4 blgp:4"


@pytest.mark.parametrize("code,faults", [
    ([FP8, "s_nop 10", "v_accvgpr_read_b32 v1, a3"], 1),
    ([FP8, "s_nop 11", "v_accvgpr_read_b32 v1, a3"], 0),
    ([FP4, "s_nop 6", "v_accvgpr_read_b32 v1, a3"], 1),
    ([FP4, "s_nop 7", "v_accvgpr_read_b32 v1, a3"], 0),
    ([FP8, "s_nop 9", "v_accvgpr_write_b32 a2, 0"], 1),
    ([FP8, "s_nop 10", "v_accvgpr_write_b32 a2, 0"], 0),
    ([FP8, FP8], 0),                                                        # the sum goes on in its registers
    ([FP8, FP8.replace("a[0:3], v40", "a[4:7], v40")], 0),                  # overwritten
    ([FP8, FP8.replace(" a[0:3], v[10", " a[4:7], v[10")], 0),              # the sum goes on in others
    ([FP8, FP8.replace("a[0:3]", "a[2:5]")], 1),                            # ... from half of it
    ([FP8, FP8.replace("v[10:13]", "a[0:3]")], 1),                          # as an operand
    ([FP8, "global_store_dwordx4 v[30:31], a[0:3], off"], 1),
    (["s_nop 7", "loop:", "v_accvgpr_read_b32 v1, a0", "s_nop 1", FP8, "s_cbranch_scc1 loop"], 1),       # around the loop
    (["s_nop 7", "loop:", "v_accvgpr_read_b32 v1, a0", "s_nop 1", FP8, "s_nop 11", "s_cbranch_scc1 loop"], 0),
    ([FP8, "s_branch there", "v_accvgpr_read_b32 v1, a0", "there:", "s_nop 15"], 0),
    (["v_mov_b32_e32 v22, 0", "s_nop 0", FP8], 1),
    (["v_mov_b32_e32 v22, 0", "s_nop 1", FP8], 0),
    (["v_lshrrev_b32_e32 v40, 8, v40", FP8], 1),                            # a scale
    (["v_accvgpr_write_b32 a1, 0", "s_nop 0", FP8], 1),                     # the sum itself
    (["v_mov_b32_e32 v22, 0", "s_cbranch_scc1 there", "s_nop 1", "there:", FP8], 1),
    (["v_mov_b32_e32 v50, 0", FP8], 0),
    (["v_cmp_gt_u32_e32 vcc, 8, v22", FP8], 0),
])
def test_the_walk_sees_planted_mistakes(code, faults):
    text = "_ZN2sg1xEv: ; @\n\t" + "\n\t".join(code + ["s_endpgm"]) + "\n\t.section\n"
    assert len(early(*_functions(text)["_ZN2sg1xEv"])[1]) == faults
