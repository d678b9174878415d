"""What the inline-assembly MFMAs of the tiles with MXFP4 weights rest on, read from
this build's own code: the compiler does not know that they are MFMAs, so it does not
keep their operands' distances.

  - A vector register that a VALU instruction writes, an operand's or a scale's, may be
    read by an MFMA two wait states later at the earliest (loads are waited for by the
    waitcnt that the compiler sets for any use).
  - The accumulators stay where they are: the loop over the steps moves none."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT
from test_ffn_asm import BUILD, OBJDUMP, operands, registers

OBJECTS = ["k_mx_bf16.hip.o", "k_mx_fp8.hip.o", "k_mx_fp4.hip.o"]
STATES = 2
VALU = re.compile(r"v_(?!mfma|cmp|nop|readfirstlane)")


def written(ins):
    ops = operands(ins)
    return registers(" ".join(ops[:2] if "_swap_" in ins else ops[:1])) if VALU.match(ins) else set()


def states(ins):
    return int(operands(ins)[0], 0) + 1 if ins.startswith("s_nop") else 1


def hazards(ins, jumps):
    """(writer, mfma) pairs with fewer than STATES wait states between them, on the paths that fall through and on those
    over one branch; jumps: {index of a target: indices of its branches}."""
    bad = []

    def back(to, left, reads, s, over):                            # what comes before ins[to]
        for b in () if over else jumps.get(to, ()):
            back(b + 1, left, reads, s, True)
        if to == 0:
            return
        if written(ins[to - 1]) & reads:
            bad.append((ins[to - 1], s))
        left -= states(ins[to - 1])
        if left > 0:
            back(to - 1, left, reads, s, over)
    for i, s in enumerate(ins):
        if s.startswith("v_mfma"):
            scaled = s.startswith("v_mfma_scale")
            back(i, STATES, set().union(*map(registers, operands(s)[1:6 if scaled else 4])), s, False)
    return bad


def kernels(path, tmp_path):
    """{kernel: (instructions, {target index: branch indices})} of one object."""
    obj = shutil.copy(path, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", obj], check=True, stdout=subprocess.DEVNULL, cwd=tmp_path)
    [code] = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", os.path.join(tmp_path, code)], check=True,
                          capture_output=True, text=True).stdout
    out = {}
    for name, body in re.findall(r"^[0-9a-f]+ <(\S*k_mx_gemm\S*)>:\n((?:[ \t].*\n)+)", text, re.M):
        ins, at, branches, start = [], {}, [], None
        for line in body.splitlines():
            s, _, addr = line.partition("//")
            if not addr:                                            # "...": zeros behind the code
                continue
            addr = int(addr.strip().split(":")[0].split()[0], 16)
            start = addr if start is None else start
            at[addr - start] = len(ins)
            t = re.search(r"<\S+\+0x([0-9a-f]+)>", line) if s.split()[0].startswith(("s_branch", "s_cbranch")) else None
            if t:
                branches.append((len(ins), int(t.group(1), 16)))
            ins.append(" ".join(s.split()))
        jumps = {}
        for i, target in branches:
            jumps.setdefault(at[target], []).append(i)
        out[name] = ins, jumps
    return out


@pytest.mark.parametrize("obj", OBJECTS)
def test_mfma_operands(obj, tmp_path):
    path = os.path.join(BUILD, obj)
    if not (os.path.exists(path) and os.path.exists(OBJDUMP)):
        pytest.skip("no objects of a build here")
    found = kernels(path, tmp_path)
    assert found
    for name, (ins, jumps) in found.items():
        mfma = [i for i, s in enumerate(ins) if s.startswith("v_mfma")]
        assert mfma, name
        assert not hazards(ins, jumps), (name, hazards(ins, jumps)[:3])
        loops = [(t, b) for t, bs in jumps.items() for b in bs if t <= b]
        main = min((b + 1 - t, t) for t, b in loops if any(t <= i <= b for i in mfma))
        assert not [s for s in ins[main[1]:sum(main)] if s.startswith("v_accvgpr")], name


def test_the_check_finds_a_near_write():
    mfma = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:3], v[4:11], a[0:3], v20, v21 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4"
    for w in ("v_mov_b32_e32 v1, 0", "v_perm_b32 v21, v1, v2, v3", "v_permlane16_swap_b32_e32 v30, v20"):
        assert hazards([w, mfma], {}) and hazards([w, "s_nop 0", mfma], {})
        assert not hazards([w, "s_nop 1", mfma], {}) and not hazards([w, "s_nop 0", "s_nop 0", mfma], {})
    loop = [mfma, "v_mov_b32_e32 v5, 0", "s_cbranch_scc1 65530"]
    assert not hazards(loop, {}) and hazards(loop, {0: [2]})
    assert not hazards(["v_mov_b32_e32 v40, 0", mfma], {})
