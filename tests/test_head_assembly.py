"""What the compiler cannot see, looked up in the code that it made.

The largest tiles' products are written out, with their sums in the
accumulation registers for good, so the compiler does not put the wait states
around them that it puts around its own: two between a vector instruction's write
of a factor and the product, and 18 between a product and another use of its sum
(more than these products' 8 passes take).  The source keeps both: factors come
from LDS reads alone, and sums are left alone for 32 states.  Here the library's
gfx950 code is read again for it.
"""
import os
import re
import struct
import subprocess
from pathlib import Path

import pytest

from test_head_ops import CSRC, native  # noqa: F401

OBJDUMP = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm" / "bin" / "llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def device_code(library):
    """The gfx950 objects in a library."""
    data, at = library.read_bytes(), -1
    while (at := data.find(MAGIC, at + 1)) >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(count if count < 16 else 0):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            name = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            if name.endswith(b"gfx950") and size:
                yield data[at + offset:at + offset + size]


def registers(text):
    """The registers that an operand names, as {(kind, number)}."""
    found = set()
    for kind, one, low, high in re.findall(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        numbers = range(int(one), int(one) + 1) if one else range(int(low), int(high) + 1)
        found |= {(kind, n) for n in numbers}
    return found


class Instruction:
    def __init__(self, text, address):
        self.name, _, rest = text.strip().partition(" ")
        operands = re.split(r",\s*(?![^\[]*\])", rest)
        self.address, self.before = address, []
        self.product = self.name.startswith("v_mfma")
        self.states = int(operands[0]) + 1 if self.name == "s_nop" else 1
        self.uses = registers(rest)
        self.factors = registers(operands[1] + "," + operands[2]) if self.product else set()
        self.writes = set()
        if self.name.startswith("v_") and not self.name.startswith("v_cmp"):
            self.writes = registers(operands[0])
            if "swap" in self.name:
                self.writes |= registers(operands[1])


def parse(lines):
    """One kernel's instructions, each with those that may come before it."""
    code, jumps = [], []
    for line in lines:
        m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+): (.*)$", line)
        if not m:
            continue
        code.append(Instruction(m[1], int(m[2], 16)))
        if code[-1].name.startswith(("s_branch", "s_cbranch")):
            to = re.search(r"<[^+>]*(?:\+0x([0-9a-f]+))?>", m[3])
            jumps.append((code[-1], int(to[1] or "0", 16)))
    start, at = code[0].address, {i.address: i for i in code}
    for a, b in zip(code, code[1:]):
        if a.name not in ("s_branch", "s_endpgm"):
            b.before.append(a)
    for jump, to in jumps:
        at[start + to].before.append(jump)
    return code


def within_states(instruction, states, seen=None):
    """What runs less than `states` wait states before an instruction."""
    for b in instruction.before:
        yield b
        if b.states < states:
            yield from within_states(b, states - b.states)


def faults(code):
    for i in code:
        if i.product:
            for b in within_states(i, 2):
                if not b.product and b.writes & i.factors:
                    yield f"{b.name} writes a factor of {i.name} at {i.address:x}"
        else:
            sums = {r for r in i.uses if r[0] == "a"}
            for b in within_states(i, 18) if sums else ():
                if b.product and b.writes & sums:
                    yield f"{i.name} at {i.address:x} uses a sum of the {b.name} at {b.address:x}"


def listing(*lines):
    return parse(f"\t{text} // {4 * n:012X}: 00000000 {to}" for n, (text, _, to) in
                 enumerate(line.partition(" -> ") for line in lines))


PRODUCT = "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]"


@pytest.mark.parametrize("lines,wrong", [
    (["v_mov_b32_e32 v4, v1", PRODUCT], 1),
    (["v_mov_b32_e32 v11, v1", "s_add_u32 s0, s0, 1", PRODUCT], 1),
    (["v_mov_b32_e32 v11, v1", "s_nop 1", PRODUCT], 0),
    (["v_mov_b32_e32 v12, v4", PRODUCT], 0),
    (["v_cmp_gt_i32_e32 vcc, s4, v5", PRODUCT], 0),
    (["ds_read_b128 v[4:7], v30 offset:16", "s_waitcnt lgkmcnt(0)", PRODUCT], 0),
    ([PRODUCT, "s_nop 15", "v_accvgpr_read_b32 v20, a3"], 1),
    ([PRODUCT, "s_nop 15", "s_nop 15", "v_accvgpr_read_b32 v20, a3"], 0),
    ([PRODUCT, "v_accvgpr_read_b32 v20, a4"], 0),
    # the jump is one state
    (["s_nop 0", PRODUCT, "v_mov_b32_e32 v4, v1", "s_cbranch_scc1 65533 -> <f+0x4>"], 1),
    ([PRODUCT, "v_swap_b32 v1, v4", "s_branch 65533 -> <f>"], 1),
    ([PRODUCT, "v_swap_b32 v1, v4", "s_nop 0", "s_branch 65533 -> <f>"], 0),
    (["s_branch 2 -> <f+0xc>", "v_mov_b32_e32 v4, v1", "s_nop 0", PRODUCT], 1),
    (["s_branch 2 -> <f+0xc>", "v_mov_b32_e32 v4, v1", "s_endpgm", PRODUCT], 0),
    (["s_cbranch_scc1 1 -> <f+0x8>", "v_mov_b32_e32 v4, v1", PRODUCT], 1)], ids=str)
def test_the_reader(lines, wrong):
    assert len(list(faults(listing(*lines)))) == wrong


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no llvm-objdump")
def test_wait_states_around_the_largest_tiles_products(tmp_path):
    kernels = 0
    for n, code in enumerate(device_code(CSRC / "libvgpu_ops.so")):
        path = tmp_path / f"{n}.o"
        path.write_bytes(code)
        out = subprocess.run([str(OBJDUMP), "-d", str(path)], capture_output=True, text=True, check=True)
        for block in re.split(r"\n(?=[0-9a-f]{16} <)", out.stdout):
            head, _, body = block.partition("\n")
            if "gemm_tile" not in head or "Li256ELi256E" not in head:
                continue
            code = parse(body.splitlines())
            assert sum(i.product and ("a", 0) in i.writes for i in code) > 0, head
            assert not (wrong := list(faults(code))), (head, wrong[:5])
            kernels += 1
    assert kernels == 12  # three types, either operand's two layouts
