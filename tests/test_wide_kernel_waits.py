"""The wide product kernels' matrix instructions and copies stand in inline
assembly, where the compiler adds no waits. Their built code is read here for
those that the hardware does not keep by itself, along every path:

  - an operand of a matrix instruction that a vector instruction wrote: two
    states before it;
  - a matrix instruction's result read or overwritten by another kind of
    instruction: eighteen (the most that any of its kind needs);
  - a scalar register of a memory access that a vector instruction wrote: five;
  - a copy to LDS after m0 was set: one.
"""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
BUILD = ROOT / "burn-deltanet_amd" / "_build"
OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
MATRIX_RESULT, MATRIX_OPERAND, SCALAR_ADDRESS = 18, 2, 5


def registers(text):
    """The registers named in an operand list, as (kind, number)."""
    out = set()
    for kind, first, last, one in re.findall(r"\b([vas])(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        for n in range(int(first or one), int(last or one) + 1):
            out.add((kind, n))
    if re.search(r"\bvcc\b", text):
        out.add(("s", "vcc"))
    if re.search(r"\bm0\b", text):
        out.add(("s", "m0"))
    return out


class Instruction:
    def __init__(self, line):
        text, _, comment = line.strip().partition("//")
        self.at = int(comment.split(":")[0], 16)
        self.op, _, operands = text.strip().partition(" ")
        parts = operands.split(",")
        self.matrix = "mfma" in self.op
        self.vector = self.op.startswith("v_") and not self.matrix
        memory = self.op.startswith(("global_", "flat_", "buffer_", "scratch_", "ds_"))
        self.store = memory and ("store" in self.op or "write" in self.op or "lds" in self.op)
        self.memory = memory
        # What stands first is written, but by stores and copies to LDS; a few
        # instructions write a second, scalar operand.
        first = 0 if self.store or not (self.vector or self.matrix or memory
                                        or self.op.startswith("s_")) else 1
        if self.vector and re.match(r"v_(add_co|sub_co|subrev_co|addc_co|subb_co|mad_u64|mad_i64|div_scale)",
                                    self.op):
            first = 2
        if self.op.startswith(("s_cmp", "s_bitcmp", "s_waitcnt", "s_nop", "s_cbranch", "s_branch",
                               "s_barrier")):
            first = 0
        self.writes = registers(",".join(parts[:first]))
        if self.op.startswith("v_cmp") and not self.op.startswith("v_cmpx"):
            self.writes |= registers(parts[0])
        self.reads = registers(",".join(parts[first:]))
        if self.op in ("v_swap_b32",):
            self.writes = self.reads = registers(operands)
        if "global_load_lds" in self.op:
            self.reads.add(("s", "m0"))
        self.states = 1 + (int(operands.split()[0]) if self.op == "s_nop" else 0)
        m = re.search(r"\+0x([0-9a-f]+)>", comment)
        self.target = int(m[1], 16) if m and self.op.startswith(("s_branch", "s_cbranch")) else None


def kernels(path):
    """{name: instructions} of a built object's wide kernels."""
    out, name, start = {}, None, 0
    listing = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", "--no-show-raw-insn", path],
                             capture_output=True, text=True, check=True).stdout
    for line in listing.splitlines():
        m = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if m:
            name, start = (m[2], int(m[1], 16)) if "gemm_wide_kernel" in m[2] else (None, 0)
            if name:
                out[name] = []
        elif name and "//" in line:
            i = Instruction(line)
            if i.target is not None:
                i.target += start
            out[name].append(i)
    return out


def predecessors(code):
    index = {c.at: n for n, c in enumerate(code)}
    before = [[] for _ in code]
    for n, c in enumerate(code):
        if n + 1 < len(code) and c.op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before[n + 1].append(n)
        if c.target is not None:
            before[index[c.target]].append(n)
    return before


def writers(code, before, n, registers, most):
    """The last writers of `registers` ahead of n, along any path, that are fewer
    than `most` wait states ahead."""
    found, seen, work = [], {}, [(p, 0, frozenset(registers)) for p in before[n]]
    while work:
        i, passed, left = work.pop()
        if passed >= most or seen.get((i, left), most) <= passed:
            continue
        seen[i, left] = passed
        if code[i].writes & left:
            found.append((code[i], passed))
            left = left - code[i].writes
        if left:
            work += [(p, passed + code[i].states, left) for p in before[i]]
    return found


def faults(code):
    before = predecessors(code)
    out = []

    def look(n, registers, most, wrong, what):
        if registers:
            out.extend(f"{what}: {i.op} at {i.at:x}, {passed} states before {code[n].op} at "
                       f"{code[n].at:x}"
                       for i, passed in writers(code, before, n, registers, most) if wrong(i))

    for n, c in enumerate(code):
        if c.matrix:
            look(n, c.reads, MATRIX_OPERAND, lambda i: i.vector, "operand")
        elif c.vector or c.memory:
            look(n, c.reads | c.writes, MATRIX_RESULT, lambda i: i.matrix, "result")
        if c.memory:
            scalars = {r for r in c.reads if r[0] == "s"}
            look(n, scalars, SCALAR_ADDRESS, lambda i: i.vector, "address")
        if "global_load_lds" in c.op:
            look(n, {("s", "m0")}, 1, lambda i: True, "m0")
    return out


def listed(*lines):
    """Instructions at consecutive addresses, for tests of the reading itself."""
    return [Instruction(f"{line} // {4 * n:012X}: 00000000") for n, line in enumerate(lines)]


@pytest.mark.parametrize("lines,bad", [
    (["v_mov_b32_e32 v1, v9", "s_nop 0",
      "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"], "operand"),
    (["v_mov_b32_e32 v1, v9", "s_nop 1",
      "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"], None),
    (["v_accvgpr_write_b32 a2, v9",
      "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"], "operand"),
    (["v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]", "s_nop 15",
      "v_accvgpr_read_b32 v9, a2"], "result"),
    (["v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]", "s_nop 15", "s_nop 15",
      "v_accvgpr_read_b32 v9, a2"], None),
    (["v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]",
      "ds_write_b128 v9, a[0:3]"], "result"),
    (["v_readfirstlane_b32 s5, v9", "s_mov_b32 m0, s9", "s_nop 0",
      "global_load_lds_dwordx4 v2, s[4:5]"], "address"),
    (["v_readfirstlane_b32 s5, v9", "s_mov_b32 m0, s9", "s_mov_b64 s[6:7], s[4:5]",
      "global_load_lds_dwordx4 v2, s[6:7]"], None),
    (["s_mov_b32 m0, s9", "global_load_lds_dwordx4 v2, s[6:7]"], "m0"),
    (["v_readlane_b32 s4, v9, 3", "global_store_dword v2, v3, s[4:5]"], "address"),
])
def test_a_missing_wait_is_seen(lines, bad):
    found = faults(listed(*lines))
    assert [f.split(":")[0] for f in found] == ([bad] if bad else [])


def test_loops_are_followed():
    code = listed("v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]", "s_nop 0",
                  "v_mov_b32_e32 v4, v9", "s_cbranch_scc1 4")
    assert not faults(code)
    code[3].target = 0
    assert [f.split(":")[0] for f in faults(code)] == ["operand"]


@pytest.mark.parametrize("name", ["gemm_bf16", "gemm_f8"])
def test_wide_kernels_wait(name, tmp_path):
    built = BUILD / f"{name}.o"
    if not built.exists() or not OBJDUMP.exists():
        pytest.skip("the library's objects are not here")
    shutil.copy(built, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", built.name], cwd=tmp_path, check=True,
                   capture_output=True)
    device, = tmp_path.glob("*gfx950")
    found = kernels(device)
    assert len(found) == (5 if name == "gemm_bf16" else 2)
    for kernel, code in found.items():
        assert sum(c.matrix for c in code) >= 128 and any("load_lds" in c.op for c in code)
        assert faults(code) == [], kernel
