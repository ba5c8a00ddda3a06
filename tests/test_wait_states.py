"""Wait states of the built kernels (CPU only): what the gfx950 compiler adds by itself between its own
instructions, but not inside inline assembly.

A vector instruction that writes a scalar register (v_readfirstlane, a compare, a carry) has to be
five wait states away from a memory instruction that reads it as an address, and a scalar write of
m0 one from a load to LDS: the hardware does not wait, and a load that comes earlier may use what the
register held before. Every instruction counts one, s_nop N counts N + 1. The listing is of
``libslime_ca.so``, as built here from the sources.
"""
import os
import re
import shutil
import subprocess

import pytest

from slime_amd import _lib, build

ADDRESS, M0 = 5, 1
MEMORY = ("global_", "buffer_", "flat_", "scratch_")
# A carry or flag as their second operand.
SECOND = re.compile(r"v_(mad_u64_u32|mad_i64_i32|add_co_|sub_co_|subrev_co_|addc_co_|subb_co_|subbrev_co_|div_scale_)")
REG = re.compile(r"s\[(\d+):(\d+)\]|s(\d+)|(vcc)(?:_lo|_hi)?")


def scalars(operand):
    """The scalar registers that an operand names."""
    m = REG.fullmatch(operand)
    if not m:
        return set()
    if m.group(4):
        return {"vcc"}
    lo = int(m.group(1) or m.group(3))
    return set(range(lo, int(m.group(2) or lo) + 1))


class Instruction:
    def __init__(self, text):
        name, _, rest = text.partition(" ")
        ops = [o for o in re.split(r"[ ,]+", rest.strip()) if o]
        self.text, self.name = text, name
        self.waits = int(ops[0], 0) + 1 if name == "s_nop" else 1
        self.valu_writes, self.reads, self.m0 = set(), set(), False
        if name.startswith("v_"):
            # The first operand, if it is scalar (v_readfirstlane, compares), or a second one that is written.
            self.valu_writes = scalars(ops[0]) if ops else set()
            if SECOND.match(name) and len(ops) > 1:
                self.valu_writes |= scalars(ops[1])
        elif name.startswith(MEMORY):
            self.reads = set().union(*map(scalars, ops)) if ops else set()
        elif name.startswith("s_"):
            self.m0 = bool(ops) and ops[0] == "m0" and not name.startswith("s_cmp")
        self.to_lds = name.startswith(MEMORY) and ("_lds_" in name or "lds" in ops)
        self.target = ops[0] if name.startswith(("s_cbranch", "s_branch")) else None
        self.ends = name in ("s_branch", "s_endpgm", "s_setpc_b64")


def too_close(listing):
    """[(function, first instruction, second, wait states)] of an llvm-objdump listing."""
    found = []
    for name, lines in _functions(listing):
        code, labels = [], {}
        for line in lines:
            label = re.match(r"^(?:[0-9a-f]+ )?<(\w+)>:", line)
            if label:
                labels[label.group(1)] = len(code)
            elif line.startswith("\t"):
                code.append(Instruction(line.split("//")[0].strip()))
        before = [[] for _ in code]  # which instructions may run just before each
        for i, x in enumerate(code):
            if not x.ends and i + 1 < len(code):
                before[i + 1].append(i)
            if x.target is not None and labels.get(x.target, len(code)) < len(code):
                before[labels[x.target]].append(i)
        for i, x in enumerate(code):
            if not x.reads and not x.to_lds:
                continue
            todo, least = [(p, 0) for p in before[i]], {}
            while todo:
                p, waits = todo.pop()
                if waits >= ADDRESS or least.get(p, ADDRESS) <= waits:
                    continue
                least[p] = waits
                y = code[p]
                if y.valu_writes & x.reads or (x.to_lds and y.m0 and waits < M0):
                    found.append((name, y.text, x.text, waits))
                todo += [(b, waits + y.waits) for b in before[p]]
    return found


def _functions(listing):
    name, lines = None, []
    for line in listing.splitlines():
        m = re.match(r"^[0-9a-f]+ <([^>]+)>:", line)
        if m and not re.fullmatch(r"L\d+", m.group(1)):
            if name:
                yield name, lines
            name, lines = m.group(1), []
        else:
            lines.append(line)
    if name:
        yield name, lines


def listings(folder):
    """The disassembly of each part of the library's device code."""
    objdump = os.path.join(os.path.dirname(os.path.realpath(build.hipcc())), "..", "llvm", "bin", "llvm-objdump")
    if not os.path.exists(objdump):
        objdump = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
    lib = os.path.join(folder, "lib.so")
    shutil.copy(_lib.LIB_PATH, lib)
    subprocess.run([objdump, "--offloading", lib], check=True, capture_output=True)
    for part in sorted(os.listdir(folder)):
        if part.endswith(build.ARCH):
            yield subprocess.run([objdump, "-d", "--symbolize-operands", "--no-show-raw-insn", os.path.join(folder, part)],
                                 check=True, capture_output=True, text=True).stdout


def test_addresses_are_settled_before_memory_instructions(tmp_path):
    loads, found = 0, []
    for text in listings(str(tmp_path)):
        loads += text.count("global_load_lds")
        found += too_close(text)
    assert loads > 1000, "the listing shows the direct loads"
    names = {}
    for name, *_ in found:
        names[name] = names.get(name, 0) + 1
    assert not found, f"{len(found)} in {len(names)} kernels, such as {found[:3]}; {names}"


@pytest.mark.parametrize("between, waits", [("", 2), ("\ts_nop 1\n", 4), ("\ts_nop 2\n", None)])
def test_listings_with_too_few_are_reported(between, waits):
    text = f"""0000000000001000 <kernel>:
\tv_readfirstlane_b32 s9, v9      // 0000: 0
{between}\ts_mov_b32 m0, s4        // 0004: 0
\ts_nop 0                         // 0008: 0
\tglobal_load_lds_dwordx4 v4, s[8:9] // 000C: 0
\ts_endpgm                        // 0014: 0
"""
    assert [w for *_, w in too_close(text)] == ([] if waits is None else [waits])


def test_branches_are_followed():
    text = """0000000000001000 <kernel>:
0000000000001000 <L0>:
\tv_cmp_lt_i32_e64 s[2:3], v0, v1
\ts_cbranch_scc0 L1
\ts_nop 4
\ts_branch L2
0000000000001020 <L1>:
\ts_nop 0
0000000000001030 <L2>:
\tglobal_load_dword v1, v0, s[2:3]
\ts_mov_b32 m0, s7
\tglobal_load_lds_dword v1, v0, s[4:5]
\ts_endpgm
"""
    assert sorted(w for *_, w in too_close(text)) == [0, 2]
