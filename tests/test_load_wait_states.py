"""The machine code of libhbt.so keeps the wait states that loads into LDS need.

The hardware does not hold such a load back for the scalar registers it reads.  Between a vector
instruction that writes one of them (``v_readfirstlane_b32``, a comparison) and a buffer instruction
that reads it there must be five wait states, and one between a scalar write of m0 and a load into
LDS.  The compiler keeps both for its own instructions and does not look into inline assembly, so
the device code is taken out of the library that was built here and every path of five wait states
that ends in a load into LDS is looked at.  Needs no device.
"""

from __future__ import annotations

import os
import re
import shutil
import struct
import subprocess

import pytest

from hybrid_training_amd import _native

OBJDUMP = shutil.which("llvm-objdump", path=os.environ.get("PATH", "") + ":/opt/rocm/llvm/bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
VALU_SGPR, SALU_M0 = 5, 1


def device_objects(path):
    """The gfx950 code objects bundled in a library."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", data, at + 24)
        entry = at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24 : entry + 24 + length]:
                yield data[at + offset : at + offset + size]
            entry += 24 + length
        at = data.find(MAGIC, at + 1)


def registers(text):
    """Scalar registers that an operand names."""
    if text in ("vcc", "m0"):
        return {text}
    if found := re.fullmatch(r"s\[(\d+):(\d+)\]", text):
        return {f"s{i}" for i in range(int(found[1]), int(found[2]) + 1)}
    return {text} if re.fullmatch(r"s\d+", text) else set()


LINE = re.compile(r"^\t(\S+)(?: (.*?))?\s*// ([0-9A-F]+):.*?(?:<(.+?)\+0x([0-9a-f]+)>|<(\S+?)>)?$")


class Instruction:
    __slots__ = ("op", "operands", "address", "target", "before")

    def __init__(self, op, operands, address, target):
        self.op, self.operands, self.address, self.target = op, operands, address, target
        self.before = []  # the instructions that may run just before it

    @property
    def states(self):
        return int(self.operands[0], 0) + 1 if self.op == "s_nop" else 1

    def written(self):
        """Scalar registers it writes: the first operand, and a vector instruction's second one (a carry)."""
        if self.op.startswith("v_cmp") and self.op.endswith("_e32"):
            return {"vcc"}
        ends = 2 if self.op.startswith(("v_add_co", "v_sub_co", "v_subrev_co", "v_addc_co", "v_subb_co", "v_div_scale",
                                        "v_mad_u64", "v_mad_i64")) else 1
        return set().union(*(registers(o) for o in self.operands[:ends])) if self.operands else set()


def functions(listing):
    """Lists of instructions with their predecessors."""
    start, body, entry = None, [], {}
    for line in listing.splitlines():
        if found := re.match(r"^([0-9a-f]+) <(.+)>:$", line):
            start, body = found[2], []
            entry[start] = (int(found[1], 16), body)
        elif start is not None and (found := LINE.match(line)):
            target = None
            if found[1].startswith(("s_branch", "s_cbranch")):
                target = (found[4] or found[6], int(found[5] or "0", 16))
            body.append(Instruction(found[1], [o.strip() for o in re.split(r",\s*|\s+", found[2] or "") if o],
                                    int(found[3], 16), target))
    for first, body in entry.values():
        by_address = {i.address: i for i in body}
        for i, instruction in enumerate(body):
            if i > 0 and body[i - 1].op not in ("s_branch", "s_endpgm", "s_setpc_b64", "s_swappc_b64"):
                instruction.before.append(body[i - 1])
            if instruction.target is not None:
                name, offset = instruction.target
                by_address[entry[name][0] + offset].before.append(instruction)
        yield body


def faults(load):
    """What is too close before a load into LDS."""
    reads = set().union(*(registers(o) for o in load.operands[1:]))
    found, work, seen = [], [(i, 0) for i in load.before], {}
    while work:
        instruction, states = work.pop()
        if states >= VALU_SGPR or seen.get(instruction, VALU_SGPR) <= states:
            continue
        seen[instruction] = states
        writes = instruction.written()
        if instruction.op.startswith("v_") and writes & reads:
            found.append(f"{instruction.op} of {sorted(writes & reads)} {states} wait states before")
        if "m0" in writes and states < SALU_M0:
            found.append(f"{instruction.op} of m0 {states} wait states before")
        work += [(i, states + instruction.states) for i in instruction.before]
    return found


def check(listing):
    loads = problems = 0
    first = None
    for body in functions(listing):
        for instruction in body:
            if instruction.op.startswith("buffer_load") and instruction.operands[-1] == "lds":
                loads += 1
                if found := faults(instruction):
                    problems += 1
                    first = first or f"{instruction.address:x}: {instruction.op} {instruction.operands}: {found}"
    return loads, problems, first


def listing(code, tmp_path):
    path = tmp_path / "device.co"
    path.write_bytes(code)
    return subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True,
                          text=True).stdout


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump on this host")
def test_loads_into_lds_keep_their_wait_states(tmp_path):
    objects = list(device_objects(_native.library()._name))
    assert objects, "no gfx950 code in the library"
    loads = 0
    for code in objects:
        if b"product_kernel" not in code and b"newton_schulz_kernel" not in code:
            continue
        found, problems, first = check(listing(code, tmp_path))
        assert problems == 0, f"{problems} of {found} loads: {first}"
        loads += found
    assert loads > 1000  # the tile products' loads, in every form of theirs


def test_the_check_sees_what_it_looks_for():
    def code(*lines):
        text = "0000000000000100 <f>:\n"
        for i, line in enumerate(lines):
            text += f"\t{line}    // {0x100 + 4 * i:012X}: 00000000\n"
        return text

    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    near = ["v_readfirstlane_b32 s4, v4", "s_mov_b32 m0, s8", "s_nop 2", load]
    far = ["v_readfirstlane_b32 s4, v4", "s_mov_b32 m0, s8", "s_nop 3", load]
    assert check(code(*near))[:2] == (1, 1) and check(code(*far))[:2] == (1, 0)
    assert check(code("v_readfirstlane_b32 s3, v4", "s_mov_b32 m0, s8", "s_nop 0", load))[:2] == (1, 0)
    assert check(code("s_mov_b32 m0, s8", load))[:2] == (1, 1)
    assert check(code("v_cmp_gt_u32_e64 s[6:7], v1, v2", "s_nop 3", load))[:2] == (1, 1)
    assert check(code("s_mov_b32 s4, s8", load))[:2] == (1, 0)
    # round a loop's back edge
    loop = "0000000000000100 <f>:\n\ts_nop 4    // 000000000100: 0\n\t" + load + "    // 000000000104: 0\n"
    loop += "\tv_readlane_b32 s5, v9, 1    // 000000000108: 0\n\ts_cbranch_scc1 65533    // 00000000010C: 0 <f+0x4>\n"
    assert check(loop)[:2] == (1, 1)
    assert check(loop.replace("v_readlane_b32 s5", "v_readlane_b32 s15"))[:2] == (1, 0)
