"""Runs the built code of a gfx950 kernel on the CPU, a wave at a time, as far as its
addresses go: what the compiler made of a kernel's bounds, which reading its source does
not show.

  - A load or store outside the buffers that the caller names, an LDS access outside the
    launch's LDS, a read past the kernel's arguments, a register that is read or written
    while a load into it is in flight: Fault.
  - Loaded values, floating point and matrix results are random numbers: no address may
    depend on them. Of v_rcp_iflag_f32 (divisions of integers) one of the two numbers
    around the quotient, at random.
  - Barriers are counted, not waited at: waves that do not depend on each other's loads.

Only the instructions that the kernels walked so far have; any other one is a Fault.
"""
import os
import re
import shutil
import struct
import subprocess

import numpy as np

from test_ffn_asm import OBJDUMP

VCC, EXEC, M0 = 106, 126, 124                                       # scalar registers; pairs, the first two
FULL = (1 << 64) - 1
LANES = np.arange(64)


class Fault(Exception):
    pass


def functions(obj, pattern, tmp_path):
    """{name: (instructions, {index of a branch: index of its target})} of an object's kernels."""
    obj = shutil.copy(obj, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", obj], check=True, stdout=subprocess.DEVNULL, cwd=tmp_path)
    [code] = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", os.path.join(tmp_path, code)], check=True, capture_output=True, text=True).stdout
    out = {}
    for name, body in re.findall(r"^[0-9a-f]+ <(\S*%s\S*)>:\n((?:[ \t].*\n)+)" % pattern, text, re.M):
        ins, at, branches, start = [], {}, [], None
        for line in body.splitlines():
            s, _, addr = line.partition("//")
            if not addr:                                            # "...": zeros behind the code
                continue
            addr = int(addr.split(":")[0], 16)
            start = addr if start is None else start
            at[addr - start] = len(ins)
            if s.split()[0].startswith(("s_branch", "s_cbranch")):
                branches.append((len(ins), int((re.search(r"<\S+?\+0x([0-9a-f]+)>", line) or re.search(r"()", "")).group(1) or "0", 16)))
            ins.append(decode(s))
        out[name] = ins, {i: at[t] for i, t in branches}
    return out


def decode(s):
    """(name, operands, modifiers)"""
    op, _, rest = s.strip().partition(" ")
    ops = [t.strip() for t in re.split(r",(?![^\[]*\])", rest)] if rest else []
    more = ""
    if ops and not op.startswith("s_waitcnt"):
        ops[-1], _, more = ops[-1].partition(" ")
    return op, ops, more


def registers(t):
    """("v" or "s", numbers) of an operand, or None; accumulators are vector registers from 256 on."""
    m = re.match(r"^[-|]*([vsa])(?:(\d+)|\[(\d+):(\d+)\])\|?$", t)
    if m:
        a, b = int(m.group(2) or m.group(3)), int(m.group(4) or m.group(2) or 0)
        up = 256 if m.group(1) == "a" else 0
        return "v" if up else m.group(1), range(a + up, b + up + 1)
    return {"vcc": ("s", range(VCC, VCC + 2)), "exec": ("s", range(EXEC, EXEC + 2)), "m0": ("s", range(M0, M0 + 1))}.get(t)


def literal(t):
    if re.match(r"^-?\d+$", t):
        return int(t) & 0xFFFFFFFF
    return int(t, 16) if t.startswith("0x") else struct.unpack("<I", struct.pack("<f", float(t)))[0]


def signed(x):
    return (x ^ 1 << 31) - (1 << 31)


COMPARE = {"lg": lambda a, b: a != b, "ne": lambda a, b: a != b, "eq": lambda a, b: a == b, "lt": lambda a, b: a < b, "le": lambda a, b: a <= b,
           "gt": lambda a, b: a > b, "ge": lambda a, b: a >= b, "ngt": lambda a, b: ~(a > b), "nlt": lambda a, b: ~(a < b)}
SCALAR = {"and": lambda a, b: a & b, "or": lambda a, b: a | b, "xor": lambda a, b: a ^ b, "andn2": lambda a, b: a & ~b,
          "lshl": lambda a, b: a << (b & 63), "lshr": lambda a, b: a >> (b & 63), "bfe": lambda a, b: a >> (b & 31) & ((1 << (b >> 16 & 127)) - 1)}
WORDS = {  # 32 bits in, 32 bits out
    "add_u32": lambda a, b: a + b, "sub_u32": lambda a, b: a - b, "subrev_u32": lambda a, b: b - a, "mul_lo_u32": lambda a, b: a * b,
    "mul_hi_u32": lambda a, b: a.astype(np.uint64) * b.astype(np.uint64) >> np.uint64(32), "and_b32": lambda a, b: a & b,
    "or_b32": lambda a, b: a | b, "xor_b32": lambda a, b: a ^ b, "lshlrev_b32": lambda a, b: b << (a & np.uint32(31)),
    "lshrrev_b32": lambda a, b: b >> (a & np.uint32(31)), "min_u32": np.minimum, "max_u32": np.maximum,
    "mul_u32_u24": lambda a, b: (a & np.uint32(0xFFFFFF)) * (b & np.uint32(0xFFFFFF)),
    "lshl_or_b32": lambda a, b, c: a << (b & np.uint32(31)) | c, "and_or_b32": lambda a, b, c: a & b | c,
    "lshl_add_u32": lambda a, b, c: (a << (b & np.uint32(31))) + c, "add_lshl_u32": lambda a, b, c: (a + b) << (c & np.uint32(31)),
    "add3_u32": lambda a, b, c: a + b + c, "or3_b32": lambda a, b, c: a | b | c,
    "bfe_u32": lambda a, b, c: a >> (b & np.uint32(31)) & ((np.uint32(1) << (c & np.uint32(31))) - np.uint32(1)),
    "mad_u32_u24": lambda a, b, c: (a & np.uint32(0xFFFFFF)) * (b & np.uint32(0xFFFFFF)) + c,
    "med3_i32": lambda a, b, c: np.sort(np.stack([a, b, c]).view(np.int32), 0)[1].view(np.uint32)}
FLOATS = {"add_f32", "sub_f32", "fma_f32", "fmac_f32", "fmaak_f32", "fmamk_f32", "max_f32", "min_f32", "rcp_f32", "exp_f32", "perm_b32", "cvt_pk_bf16_f32"}
BYTES = {"dwordx4": 16, "dwordx2": 8, "dword": 4, "ushort": 2, "short_d16_hi": 2, "short": 2}


class Wave:
    """One wave of a workgroup; buffers: {name: (address, bytes, written)}; args: the kernel's argument bytes, its blocks' count
    behind them; lds: bytes; stores: {address: number of stores}; based: a buffer descriptor's base has to be in a buffer also where
    none of its loads is."""

    def __init__(self, code, args, buffers, lds, wave, block, rng, stores, based=True):
        self.based = based
        (self.ins, self.jumps), self.args, self.buffers, self.lds, self.rng, self.stores = code, args, buffers, lds, rng, stores
        self.s = [0] * 128
        self.s[0], self.s[1], self.s[2], self.s[3] = 0x1000, 0x77, *block
        self.s[EXEC] = self.s[EXEC + 1] = 0xFFFFFFFF
        self.v = rng.integers(0, 1 << 32, (512, 64), dtype=np.uint32)
        self.v[0] = 64 * wave + LANES
        self.scc, self.barriers = False, 0
        self.loads, self.others = [], []                            # in flight: registers of vmcnt's, (kind, registers) of lgkmcnt's

    # operands
    def pair(self, r):
        return self.s[r] | self.s[r + 1] << 32

    def put_pair(self, r, x):
        self.s[r], self.s[r + 1] = x & 0xFFFFFFFF, x >> 32 & 0xFFFFFFFF

    def scalar_of(self, t, wide=False):
        r = registers(t)
        if r:
            return self.pair(r[1][0]) if wide else self.s[r[1][0]]
        x = literal(t)
        return x | (0xFFFFFFFF << 32 if t.startswith("-") else 0) if wide else x

    def words(self, t):
        if t.startswith("-") and registers(t):
            return self.words(t[1:]) ^ np.uint32(1 << 31)
        r = registers(t)
        return self.v[r[1][0]] if r and r[0] == "v" else np.full(64, self.s[r[1][0]] if r else literal(t), np.uint32)

    def pairs(self, t):
        r = registers(t)
        if r and r[0] == "v":
            return self.v[r[1][0]].astype(np.uint64) | self.v[r[1][1]].astype(np.uint64) << np.uint64(32)
        return np.full(64, self.pair(r[1][0]) if r else literal(t), np.uint64)

    def put(self, r, x):
        self.v[r] = np.where(self.live, np.asarray(x).astype(np.uint64).astype(np.uint32) if np.asarray(x).dtype != np.uint32 else x, self.v[r])

    def put_pairs(self, t, x):
        r = registers(t)[1]
        self.put(r[0], (x & np.uint64(0xFFFFFFFF)).astype(np.uint32))
        self.put(r[1], (x >> np.uint64(32)).astype(np.uint32))

    def put_mask(self, t, m):
        self.put_pair(registers(t)[1][0], sum(1 << int(i) for i in np.nonzero(m & self.live)[0]))

    def random(self, t):
        for r in registers(t)[1]:
            self.put(r, self.rng.integers(0, 1 << 32, 64, dtype=np.uint32))

    # memory
    def access(self, addresses, size, write=False):
        for a in (int(a) for a in np.unique(addresses)):
            if not any(b <= a and a + size <= b + n and (w or not write) for b, n, w in self.buffers.values()):
                near = ["%s%+d of %d" % (k, a - b, n) for k, (b, n, w) in self.buffers.items() if abs(a - b) < 1 << 36]
                raise Fault("%d bytes at %x: %s" % (size, a, near))
            if write:
                self.stores[a] = self.stores.get(a, 0) + 1

    def in_lds(self, addresses, size):
        a = addresses[self.live].astype(np.int64)
        if len(a) and (a.max() + size > self.lds or (a % size).any()):
            raise Fault("%d bytes of LDS at %d of %d" % (size, a.max(), self.lds))

    # a run
    def run(self, most=1000000):
        at = 0
        for _ in range(most):
            op, ops, more = self.ins[at]
            try:
                if op == "s_endpgm":
                    return
                to = self.step(op, ops, more, at)
            except Fault as f:
                raise Fault("%s\n  instruction %d: %s %s %s" % (f, at, op, ", ".join(ops), more)) from None
            at = at + 1 if to is None else to
        raise Fault("no end")

    def step(self, op, ops, more, at):
        if op == "s_barrier":
            self.barriers += 1
        elif op == "s_waitcnt":
            for kind, n in re.findall(r"(vmcnt|lgkmcnt)\((\d+)\)", " ".join(ops)):
                if kind == "vmcnt":
                    self.loads = self.loads[max(0, len(self.loads) - int(n)):]
                elif int(n) == 0 or not any(k == "s" for k, _ in self.others):   # LDS answers in order, scalar loads in any
                    self.others = self.others[max(0, len(self.others) - int(n)):]
        elif op == "s_nop":
            pass
        else:
            self.not_in_flight(op, ops + ["vcc"] * ("vcc" in op))
            if "branch" in op:
                how = {"s_branch": True, "s_cbranch_scc0": not self.scc, "s_cbranch_scc1": self.scc, "s_cbranch_vccz": not self.pair(VCC),
                       "s_cbranch_vccnz": self.pair(VCC), "s_cbranch_execz": not self.pair(EXEC), "s_cbranch_execnz": self.pair(EXEC)}
                return self.jumps[at] if how[op] else None
            self.scalar(op, ops) if op.startswith("s_") else self.vector(op, ops, more)

    def not_in_flight(self, op, ops):
        """A load may be aimed at registers that another one is on its way to: they come in order."""
        if self.loads or self.others:
            mine = {(r[0], k) for r in map(registers, ops[1:] if op.startswith(("buffer_load", "global_load")) else ops) if r for k in r[1]}
            for d in self.loads + [d for _, d in self.others]:
                if d & mine:
                    raise Fault("a load into %s is in flight" % sorted(d & mine))

    def scalar(self, op, t):
        if op.startswith("s_load_dword"):
            n, at = int(op.partition("x")[2] or 1), self.scalar_of(t[1], True) + literal(t[2]) - 0x7700001000
            if at < 0 or at + 4 * n > len(self.args):
                raise Fault("argument %x" % at)
            r = registers(t[0])[1]
            self.s[r[0]:r[0] + n] = struct.unpack_from("<%dI" % n, self.args, at)
            self.others.append(("s", {("s", k) for k in r}))
            return
        name, _, kind = op[2:].rpartition("_")
        wide = kind.endswith("64")
        if name in ("bitcmp0", "bitcmp1"):
            self.scc = self.scalar_of(t[0]) >> (self.scalar_of(t[1]) & 31) & 1 == int(name[-1])
            return
        if name.startswith("cmp"):
            a, b = self.scalar_of(t[0], wide), self.scalar_of(t[1], wide)
            if name.startswith("cmpk"):
                b = b & 0xFFFF | (0xFFFF0000 if kind == "i32" and b & 0x8000 else 0)
            a, b = (signed(a), signed(b)) if kind == "i32" else (a, b)
            self.scc = COMPARE[name.rpartition("_")[2]](a, b)
            return
        d = registers(t[0])[1][0]
        if name in ("and_saveexec", "andn2_saveexec"):
            old = self.pair(EXEC)
            self.put_pair(EXEC, self.scalar_of(t[1], True) & (old if name == "and_saveexec" else ~old))
            self.put_pair(d, old)
            self.scc = self.pair(EXEC) != 0
            return
        a = self.scalar_of(t[1], wide)
        b = self.scalar_of(t[2], wide) if len(t) > 2 else 0
        if name in ("movk", "addk", "mulk"):
            a = (a & 0xFFFF) - (0x10000 if a & 0x8000 else 0)
        carry = None
        if name in ("mov", "movk"):
            x = a
        elif name == "cselect":
            x = a if self.scc else b
        elif name == "mul":
            x = a * b
        elif name == "mul_hi":
            x = a * b >> 32
        elif name in ("add", "addc"):
            x = a + b + (int(self.scc) if name == "addc" else 0)
            carry = x >> 32 != 0
        elif name == "addk":
            x, carry = self.s[d] + a, False
        elif name == "mulk":
            x = self.s[d] * a
        elif name in ("sub", "subb"):
            b += int(self.scc) if name == "subb" else 0
            x, carry = a - b, b > a
        elif name in ("min", "max"):
            u, w = (signed(a), signed(b)) if kind == "i32" else (a, b)
            x = (min if name == "min" else max)(u, w)
            carry = u == x
        elif name in SCALAR:
            x = SCALAR[name](a, b) & (FULL if wide else 0xFFFFFFFF)
            carry = x != 0
        else:
            raise Fault("unknown")
        self.scc = self.scc if carry is None else carry
        if wide:
            self.put_pair(d, x)
        else:
            self.s[d] = x & 0xFFFFFFFF

    def vector(self, op, t, more):
        mask = self.pair(EXEC)
        self.live = live = np.array([mask >> i & 1 for i in range(64)], bool) if mask != FULL else np.ones(64, bool)
        m = re.search(r"offset:(-?\d+)", more)
        offset = int(m.group(1)) if m else 0
        if op.startswith("global_"):
            _, kind, width = op.split("_", 2)
            if t[2] != "off":
                raise Fault("unknown")
            a = self.pairs(t[1] if kind == "load" else t[0])[live] + np.uint64(offset & FULL)
            self.access(a, BYTES[width], kind == "store")
            if kind == "load":
                self.random(t[0])
            self.loads.append({("v", k) for k in registers(t[0])[1]} if kind == "load" else set())
            return
        if op.startswith("buffer_load_"):
            to_lds = "lds" in more.split()                          # lane after lane from m0 on
            t = ["m0"] + t if to_lds else t
            if more.split() != ["offen"] + ["lds"] * to_lds or t[3] != "0":
                raise Fault("unknown")
            r = registers(t[2])[1][0]
            base, records = self.s[r] | (self.s[r + 1] & 0xFFFF) << 32, self.s[r + 2]
            if self.s[r + 1] >> 16 or self.s[r + 3] != 0x20000:
                raise Fault("descriptor")
            if self.based and not any(b <= base < b + n for b, n, _ in self.buffers.values()):
                raise Fault("a descriptor's base, %x, is in no buffer" % base)
            o = self.words(t[1]).astype(np.int64)
            self.access(base + o[live & (o < records)], BYTES[op[12:]])
            if to_lds:
                self.in_lds(np.uint32(self.s[M0] + BYTES[op[12:]] * LANES), BYTES[op[12:]])
                self.loads.append(set())
            else:
                self.random(t[0])
                self.loads.append({("v", k) for k in registers(t[0])[1]})
            return
        if op.startswith("ds_"):
            if op == "ds_write_b128":
                self.in_lds(self.words(t[0]) + np.uint32(offset), 16)
            elif op == "ds_read_b128":
                self.in_lds(self.words(t[1]) + np.uint32(offset), 16)
            elif op.startswith("ds_read2"):
                n = 8 if op.endswith("b64") else 4
                for o in ("offset0", "offset1"):
                    o = re.search(o + r":(\d+)", more)
                    self.in_lds(self.words(t[1]) + np.uint32(int(o.group(1)) * n * (64 if "st64" in op else 1) if o else 0), n)
            elif op in ("ds_read_b32", "ds_read_b64"):
                self.in_lds(self.words(t[1]) + np.uint32(offset), int(op[-2:]) // 8)
            else:
                raise Fault("unknown")
            if op.startswith("ds_read"):
                self.random(t[0])
            self.others.append(("lds", {("v", k) for k in registers(t[0])[1]} if op.startswith("ds_read") else set()))
            return
        name = re.sub(r"_e(32|64)$", "", op[2:])
        if name == "readfirstlane_b32":
            self.s[registers(t[0])[1][0]] = int(self.words(t[1])[int(np.nonzero(live)[0][0]) if live.any() else 0])
        elif name.startswith(("mfma", "accvgpr", "cvt_scalef32")) or name.endswith("_sdwa") or name in FLOATS:
            self.random(t[0])
        elif name.startswith("permlane"):
            self.random(t[0])
            self.random(t[1])
        elif name.startswith("cmp_"):
            how, _, kind = name[4:].rpartition("_")
            a, b = (self.pairs(t[1]), self.pairs(t[2])) if kind.endswith("64") else (self.words(t[1]), self.words(t[2]))
            if kind in ("f32", "i32"):
                a, b = a.view(kind.replace("f", "float").replace("i", "int")), b.view(kind.replace("f", "float").replace("i", "int"))
            with np.errstate(invalid="ignore"):
                self.put_mask(t[0], COMPARE[how](a, b))
        elif name == "mad_u64_u32":
            x = [int(a) * int(b) + int(c) for a, b, c in zip(self.words(t[2]), self.words(t[3]), self.pairs(t[4]))]
            self.put_mask(t[1], np.array([v > FULL for v in x]))
            self.put_pairs(t[0], np.array([v & FULL for v in x], np.uint64))
        elif name == "lshl_add_u64":
            self.put_pairs(t[0], (self.pairs(t[1]) << np.uint64(self.scalar_of(t[2]))) + self.pairs(t[3]))
        elif name == "lshlrev_b64":
            self.put_pairs(t[0], self.pairs(t[2]) << np.uint64(self.scalar_of(t[1])))
        elif name == "mov_b64":
            self.put_pairs(t[0], self.pairs(t[1]))
        elif name == "mov_b32":
            self.put(registers(t[0])[1][0], self.words(t[1]))
        elif name == "cndmask_b32":
            m = self.pair(registers(t[3])[1][0])
            self.put(registers(t[0])[1][0], np.where([m >> i & 1 for i in range(64)], self.words(t[2]), self.words(t[1])))
        elif name == "bitop3_b32":
            table, x = int(re.search(r"bitop3:(\w+)", more).group(1), 0), np.zeros(64, np.uint32)
            a, b, c = (self.words(k) for k in t[1:])
            for i in range(8):
                if table >> i & 1:
                    x |= (a if i & 4 else ~a) & (b if i & 2 else ~b) & (c if i & 1 else ~c)
            self.put(registers(t[0])[1][0], x)
        elif name == "mad_i32_i24":
            a, b = ((self.words(k).astype(np.int64) & 0xFFFFFF ^ 0x800000) - 0x800000 for k in t[1:3])
            self.put(registers(t[0])[1][0], ((a * b + self.words(t[3])) & 0xFFFFFFFF).astype(np.uint32))
        elif name == "rcp_iflag_f32":
            with np.errstate(all="ignore"):
                q = 1.0 / self.words(t[1]).view(np.float32).astype(np.float64)
                f = q.astype(np.float32)
            low = np.where(f <= q, f, np.nextafter(f, np.float32(0)))
            self.put(registers(t[0])[1][0], (low if self.rng.random() < 0.5 else np.nextafter(low, np.float32(np.inf))).astype(np.float32).view(np.uint32))
        elif name == "mul_f32":
            with np.errstate(all="ignore"):
                self.put(registers(t[0])[1][0], (self.words(t[1]).view(np.float32) * self.words(t[2]).view(np.float32)).view(np.uint32))
        elif name in ("cvt_f32_u32", "cvt_f32_ubyte0"):
            x = self.words(t[1]) & np.uint32(255 if name.endswith("0") else 0xFFFFFFFF)
            self.put(registers(t[0])[1][0], x.astype(np.float32).view(np.uint32))
        elif name == "cvt_u32_f32":
            f = np.nan_to_num(self.words(t[1]).view(np.float32).astype(np.float64))
            self.put(registers(t[0])[1][0], np.clip(f, 0, 2.0 ** 32 - 1).astype(np.uint32))
        elif name in WORDS and not more:
            self.put(registers(t[0])[1][0], WORDS[name](*(self.words(k) for k in t[1:])))
        else:
            raise Fault("unknown")
