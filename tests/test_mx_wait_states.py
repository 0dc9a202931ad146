"""Wait states in the compiled microscaled products.  The compiler keeps them
between its own instructions but does not look into inline assembly, so the
whole gfx950 listing is walked: from every vector instruction along the control
flow to those that need its result, or its operands' registers, not too soon.

The distances are the compiler's own for gfx950 (an instruction counts one,
s_nop n counts n + 1):
  vector write of VCC or an SGPR        -> vector read of it                   2
  vector write of a VGPR                -> DPP read of it                      2
  vector write of a VGPR                -> matrix instruction reads it         2
  matrix instruction of four passes (4- and 6-bit operands) reads a VGPR as C
                                        -> vector write of it                  3
"""
import re
import shutil
import subprocess

import pytest

from qw3_amd import build

REG = re.compile(r"\b(vcc(?:_lo|_hi)?|[vsa]\d+|[vsa]\[\d+:\d+\])(?![\w\[])")


def registers(text):
    """Every register that the operands name; VCC as one."""
    out = set()
    for r in REG.findall(text):
        if r.startswith("vcc"):
            out.add("vcc")
        elif "[" in r:
            lo, hi = map(int, r[2:-1].split(":"))
            out.update(f"{r[0]}{i}" for i in range(lo, hi + 1))
        else:
            out.add(r)
    return out


class Instruction:
    def __init__(self, line, at):
        self.at, self.text = at, line
        self.op, _, rest = line.partition(" ")
        args = [a.strip() for a in rest.split(",")]
        self.valu = self.op.startswith("v_")
        self.mfma = self.op.startswith("v_mfma")
        self.dpp = "_dpp" in self.op or "quad_perm" in line or "row_" in line
        self.states = int(args[0], 0) + 1 if self.op == "s_nop" else 1
        self.branch = args[0] if self.op.startswith(("s_branch", "s_cbranch")) else None
        self.ends = self.op in ("s_branch", "s_endpgm", "s_setpc_b64")
        n_out = 2 if "_co_" in self.op or self.op.startswith(("v_div_scale", "v_swap", "v_mad_u64", "v_mad_i64")) else 1
        if not self.valu or self.op == "v_nop":
            self.writes, self.reads, self.dpp_reads, self.c_reads = set(), set(), set(), set()
            return
        self.writes = registers(",".join(args[:n_out]))
        self.reads = registers(",".join(args[n_out:]))
        if self.op.startswith("v_swap"):
            self.reads |= self.writes
        self.dpp_reads = registers(args[1]) if self.dpp else set()       # DPP moves the first source
        self.c_reads = registers(args[3]) - self.writes if self.mfma else set()


def parse(listing):
    """Instructions in order, and the labels' places among them."""
    code, labels = [], {}
    for line in listing.splitlines():
        line = line.split(";")[0].split("//")[0].strip()
        if m := re.match(r"([.\w$]+):$", line):
            labels[m.group(1)] = len(code)
        elif re.match(r"(v|s|ds|global|flat|scratch|buffer)_\w+", line):
            code.append(Instruction(line, len(code)))
    return code, labels


def too_early(code, labels):
    """(first, second, kind) of every pair that is closer than it may be."""
    found = []

    def walk(first, kinds):
        """Instructions behind `first` with the wait states between, along the control flow."""
        most = max(n for _, _, n, _ in kinds)
        todo, seen = [(first.at + 1, 0)] if not first.ends else [], set()
        while todo:
            at, between = todo.pop()
            if at >= len(code) or between >= most or (at, between) in seen:
                continue
            seen.add((at, between))
            i = code[at]
            for kind, regs, need, touches in kinds:
                if between < need and regs & touches(i):
                    found.append((first.text, i.text, kind))
            if i.branch in labels:
                todo.append((labels[i.branch], between + i.states))
            if not i.ends:
                todo.append((at + 1, between + i.states))

    for i in code:
        if not i.valu:
            continue
        sgprs = {r for r in i.writes if r == "vcc" or r[0] == "s"}
        vgprs = {r for r in i.writes if r[0] == "v" and r != "vcc"}
        kinds = []
        if sgprs:
            kinds.append(("mask or scalar read", sgprs, 2, lambda j: j.reads if j.valu else set()))
        if vgprs and not i.mfma:
            kinds.append(("DPP read", vgprs, 2, lambda j: j.dpp_reads))
            kinds.append(("matrix operand", vgprs, 2, lambda j: j.reads if j.mfma else set()))
        if i.c_reads:
            kinds.append(("C overwritten", i.c_reads, 3, lambda j: j.writes if j.valu and not j.mfma else set()))
        if kinds:
            walk(i, kinds)
    return found


def test_the_walk():
    """The walk itself: each kind, at its distance and one short of it, and over a loop's end."""
    pairs = [("v_cmp_eq_u32_e32 vcc, 0, v1", "v_cndmask_b32_dpp v2, v3, v4, vcc quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf", 2),
             ("v_cmp_eq_u32_e64 s[4:5], 0, v1", "v_cndmask_b32_e64 v2, v3, v4, s[4:5]", 2),
             ("v_add_u32_e32 v3, v1, v2", "v_mov_b32_dpp v2, v3 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf", 2),
             ("v_add_u32_e32 v6, v1, v2", "v_mfma_scale_f32_16x16x128_f8f6f4 v[20:23], v[4:7], v[8:11], v[12:15], v16, v17", 2),
             ("v_mfma_scale_f32_16x16x128_f8f6f4 v[20:23], v[4:7], v[8:11], v[12:15], v16, v17", "v_mov_b32_e32 v13, v40", 3)]
    for first, second, need in pairs:
        for gap in range(need + 1):
            between = [] if gap == 0 else [f"s_nop {gap - 1}"]
            code, labels = parse("\n".join([first, *between, second]))
            assert bool(too_early(code, labels)) == (gap < need), (first, gap)
    loop = [".L1:", pairs[0][1], "v_mov_b32_e32 v30, v31", "v_mov_b32_e32 v32, v31", pairs[0][0], "s_cbranch_scc1 .L1"]
    assert too_early(*parse("\n".join(loop)))
    assert not too_early(*parse("\n".join(loop[:-1] + ["s_nop 0"] + loop[-1:])))
    code, labels = parse("v_mov_b32_e32 v3, v1\ns_nop 0\nv_cndmask_b32_dpp v2, v4, v3, vcc quad_perm:[1,0,3,2]")
    assert not too_early(code, labels), "only the first source goes through DPP"


def test_wait_states(tmp_path):
    if shutil.which(build.HIPCC) is None:
        pytest.skip("no hipcc")
    out = tmp_path / "mx_matmul.s"
    flags = [f for f in build.HIP_FLAGS if f != "-fPIC"]
    subprocess.run([build.HIPCC, *flags, "-x", "hip", "-S", "--offload-device-only", str(build.CSRC / "kernels/mx_matmul.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    code, labels = parse(out.read_text())
    assert sum(i.mfma for i in code) > 1000 and any(i.dpp for i in code), "the products' listing"
    found = too_early(code, labels)
    assert not found, f"{len(found)} pairs, such as {found[0]}"
