"""What the tiled dense feed-forward kernel's inline-assembly MFMAs rest on,
read from this build's own code: the compiler does not know that they are
MFMAs, so it does not keep their operands' distances.

  - A vector register that a VALU instruction writes may be read by an MFMA
    two instructions later at the earliest (loads are waited for by the
    waitcnt that the compiler sets for any use).
  - The accumulators stay where they are: the loop over the stages moves none."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
BUILD = os.path.join(ROOT, "apus-glm5.3-flash_amd", "_build")
OBJECTS = ["k_ffn_nt.hip.o", "k_ffn_nt8.hip.o", "k_ffn_bwd.hip.o", "k_ffn_grads.hip.o"]


def registers(text):
    out = {(k, i) for k, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text) for i in range(int(a), int(b) + 1)}
    return out | {(k, int(a)) for k, a in re.findall(r"\b([va])(\d+)\b", text)}


def operands(ins):
    return ins.split(None, 1)[1].split(", ") if " " in ins else []


def hazards(ins, jumps):
    """(writer, mfma) pairs that are too near; jumps: {index of a target: indices of its branches}."""
    bad = []
    for i, s in enumerate(ins):
        if not s.startswith("v_mfma"):
            continue
        reads = set().union(*map(registers, operands(s)[1:4]))
        before = {j for d in (1, 2) for j in [i - d] if j >= 0}
        for d in (0, 1):                                            # over a branch to this one or the one before
            for b in jumps.get(i - d, ()):
                before |= {b - k for k in range(0, 2 - d) if b - k >= 0}
        for j in before:
            w = ins[j]
            if re.match(r"v_(?!mfma|cmp|nop|readfirstlane)", w) and registers(operands(w)[0]) & reads:
                bad.append((w, s))
    return bad


def kernels(path, tmp_path):
    """{kernel: (instructions, {target index: branch indices})} of one object."""
    obj = shutil.copy(path, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", obj], check=True, stdout=subprocess.DEVNULL, cwd=tmp_path)
    code = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    assert len(code) == 1
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", os.path.join(tmp_path, code[0])], check=True,
                          capture_output=True, text=True).stdout
    out = {}
    for name, body in re.findall(r"^[0-9a-f]+ <(\S*k_ffn_g(?:emm|rads)\S*)>:\n((?:[ \t].*\n)+)", text, re.M):
        start, ins, at, branches = None, [], {}, []
        for line in body.splitlines():
            s, _, addr = line.partition("//")
            if not addr:                                            # "...": zeros behind the code
                continue
            s, addr = " ".join(s.split()), int(addr.strip().split(":")[0].split()[0], 16)
            start = addr if start is None else start
            at[addr - start] = len(ins)
            t = re.search(r"<\S+\+0x([0-9a-f]+)>", line) if s.startswith(("s_branch", "s_cbranch")) else None
            if t:
                branches.append((len(ins), int(t.group(1), 16)))
            ins.append(s)
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
        assert sum(s.startswith("v_mfma") for s in ins) > 0, name
        assert not hazards(ins, jumps), (name, hazards(ins, jumps)[:3])
        loops = [(t, b) for t, bs in jumps.items() for b in bs if t <= b]
        main = min((b + 1 - t, t) for t, b in loops if any(s.startswith("v_mfma") for s in ins[t:b + 1]))
        assert not [s for s in ins[main[1]:sum(main)] if s.startswith("v_accvgpr")], name


def test_the_check_finds_a_near_write():
    far = ["v_mov_b32_e32 v1, 0", "s_nop 0", "s_nop 0", "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"]
    assert not hazards(far, {})
    assert hazards(far[:2] + far[3:], {}) and hazards(far[:1] + far[3:], {})
    loop = far[3:] + ["v_mov_b32_e32 v5, 0", "s_cbranch_scc1 65530"]
    assert not hazards(loop, {}) and hazards(loop, {0: [2]})
    assert not hazards(["v_mov_b32_e32 v9, 0"] + far[3:], {})
