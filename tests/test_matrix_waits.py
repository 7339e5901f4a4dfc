"""Reads the block-scaled product's kernels as they were built: what a matrix
instruction writes is there some cycles later, and the compiler has to leave them
before the first other instruction that reads it, on every path, branches and loops'
exits included.  No GPU."""

import os
import re
import shutil
import subprocess

import pytest

import __graft_entry__ as entry  # noqa: F401  (puts the package on the path)

OBJDUMP = shutil.which("llvm-objdump", path=os.environ["PATH"] + ":/opt/rocm/llvm/bin")
# wait states before a sum may be read, of the matrix instructions in use
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x128_f8f6f4": 12,
         "v_mfma_scale_f32_16x16x128_f8f6f4": 12}
# instructions whose first operand is read, not written
STORES = ("ds_write", "global_store", "v_cmp")


def registers(operand):
    """{(file, number)} of a vector register operand."""
    m = re.match(r"[-|]*([va])(?:\[(\d+):(\d+)\]|(\d+))", operand.strip())
    if not m:
        return frozenset()
    first = int(m.group(2) or m.group(4))
    return frozenset((m.group(1), i) for i in range(first, int(m.group(3) or first) + 1))


class Instruction:
    def __init__(self, text):
        self.name, _, rest = text.partition(" ")
        operands = [registers(o) for o in rest.split(",")] if rest.strip() else []
        vector = self.name.startswith(("v_", "ds_", "global_", "buffer_"))
        stores = self.name.startswith(STORES)
        self.states = int(rest.strip(), 0) + 1 if self.name == "s_nop" else 1
        self.matrix = self.name.startswith("v_mfma")
        self.writes = operands[0] if vector and operands and not stores else frozenset()
        read = operands if stores else operands[1:]
        if self.name.startswith(("v_fmac", "v_cvt_pk", "v_cvt_scale")):   # may keep a part of it
            read = operands
        self.reads = frozenset().union(*read) if vector else frozenset()
        self.target = None


def parsed(lines):
    """Instructions of one function's listing; branch targets as indexes."""
    code, at = [], {}
    for line in lines:
        m = re.match(r"\s+(\S.*?)\s*//\s*([0-9A-F]+):(.*)", line)
        if m:
            i = Instruction(m.group(1))
            at[int(m.group(2), 16)] = len(code)
            if i.name.startswith(("s_cbranch", "s_branch")):
                offset = re.search(r"\+0x([0-9a-f]+)>", m.group(3))
                i.target = int(offset.group(1), 16) if offset else 0
            code.append(i)
    start = min(at)
    for i in code:
        if i.target is not None:
            i.target = at[start + i.target]
    return code


def nearest_reader(code, i, limit):
    """(wait states, whether a branch lies between) of the first reader of what matrix instruction
    i writes that comes before `limit`, on any path; None without one."""
    found, seen = [], set()
    todo = [(i + 1, 0, False, code[i].writes)]
    while todo:
        j, states, branched, live = todo.pop()
        while j < len(code) and states < limit and live:
            if (j, states, branched, live) in seen:
                break
            seen.add((j, states, branched, live))
            c = code[j]
            if not c.matrix and c.reads & live:
                found.append((states, branched))
                break
            live = live - c.writes
            if c.target is not None:
                todo.append((c.target, states + 1, True, live))
                branched = True
                if c.name == "s_branch":
                    break
            elif c.name == "s_endpgm":
                break
            states += c.states
            j += 1
    return min(found) if found else None


def functions(listing):
    out, name = {}, None
    for line in listing.splitlines():
        m = re.match(r"[0-9a-f]+ <(\S+)>:", line)
        if m:
            name = m.group(1)
            out[name] = []
        elif name:
            out[name].append(line)
    return out


LISTING = """
\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], 0 // 000000000100: D3B50022 0202B522
\ts_nop 3 // 000000000108: BF800003
\ts_cbranch_scc1 2 // 00000000010C: BF850002 <f+0x18>
\ts_nop 7 // 000000000110: BF800007
\tv_mov_b32_e32 v5, v2 // 000000000114: 7E0A0302
\ts_nop {0} // 000000000118: BF800000
\tds_write_b128 v9, v[0:3] // 00000000011C: D9BE0000 00000009
\ts_endpgm // 000000000124: BF810000
"""


@pytest.mark.parametrize("nop,want", [(0, (6, True)), (1, (7, True)), (2, None)])
def test_the_reading_follows_branches(nop, want):
    """Planted: across a branch 4 + 1 + 1 + nop states after the product; without it 13."""
    code = parsed(LISTING.format(nop).splitlines())
    assert nearest_reader(code, 0, 8) == want
    assert nearest_reader(code, 0, 40) == min([(6 + nop, True), (13, True)])


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_sums_are_read_when_they_are_there(tmp_path):
    from cases.block_matmul import op
    from framework import loader
    path = loader.library_path(op.LIB_NAME, op.KERNEL_DIR)
    if not os.path.exists(path):
        loader.build_library(op.LIB_NAME, op.SOURCES, op.KERNEL_DIR)
    shutil.copy(path, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True,
                   capture_output=True)
    kernel, = [f for f in os.listdir(tmp_path) if "gfx950" in f]
    listing = subprocess.run([OBJDUMP, "-d", "--no-leading-headers", kernel], cwd=tmp_path,
                             check=True, capture_output=True, text=True).stdout
    products = straight = 0
    for name, lines in functions(listing).items():
        code = parsed(lines) if any("v_mfma" in line for line in lines) else []
        for i, c in enumerate(code):
            if c.matrix:
                products += 1
                assert nearest_reader(code, i, WAITS[c.name]) is None, f"{name}: product {i}"
                straight += nearest_reader(code, i, WAITS[c.name] + 1) is not None
    # each kind of product has readers right behind the wait: it is not longer than needed
    assert products > 1000 and straight > 100
