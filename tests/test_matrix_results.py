"""Results of the matrix cores are read late enough on every way through the delta rule's kernels, loops and branches taken included.  The
hardware does not hold such a read back and the compiler's own count is not relied on for ways over a branch: what is checked is the
generated code, in the library as it was built."""
import os
import re
import struct
import subprocess

import pytest

from nvllm_amd import capi
from tests.test_kernel_registers import MAGIC

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# Instructions (s_nop n: n + 1) that lie between a product and what first reads its result, or writes over it: what the compiler leaves in
# straight code.
WAIT = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10}


def registers(text):
    out = set()
    for a, b, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= {int(one)} if one else set(range(int(a), int(b) + 1))
    return out


class Step:
    """An instruction: registers that it reads, adds to (a product's sums, which follow one another without a wait), writes; where it goes on."""

    def __init__(self, text, at, index, target):
        self.text, self.op = text, text.split()[0]
        parts = text[len(self.op):].split(",")
        self.product = self.op.startswith("v_mfma")
        self.adds = registers(parts[3]) if self.product else set()
        reads_only = self.op.startswith(("ds_write", "buffer_store", "global_store", "scratch_store", "v_cmp", "s_"))
        both = "swap" in self.op
        self.writes = set() if reads_only or self.op.startswith(("v_readlane", "v_readfirstlane")) else registers(",".join(parts[:2]) if both else parts[0])
        self.reads = registers(",".join(parts)) if reads_only or both else registers(",".join(parts[1:3])) if self.product else registers(",".join(parts[1:]))
        self.takes = int(parts[0]) + 1 if self.op == "s_nop" else 1
        self.next = [] if self.op in ("s_endpgm", "s_branch") else [index + 1]
        if target is not None:
            self.next.append(target)


def parse(listing):
    """name -> steps of every kernel of a disassembly"""
    kernels, steps, name, start = {}, [], None, 0
    for line in listing.split("\n"):
        head = re.match(r"^([0-9a-f]+) <(\S+)>:$", line)
        if head:
            name, start = head[2], int(head[1], 16)
            kernels[name] = steps = []
            continue
        m = re.match(r"^\t(.*?)\s*// ([0-9A-Fa-f]+):(.*)$", line)
        if m and name:
            steps.append((int(m[2], 16), m[1].strip(), m[3], start))
    out = {}
    for name, lines in kernels.items():
        index = {at: i for i, (at, _, _, _) in enumerate(lines)}
        out[name] = []
        for i, (at, text, rest, start) in enumerate(lines):
            target = None
            if text.startswith(("s_cbranch", "s_branch")):
                off = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>", rest)
                target = index[start + int(off[1] or "0", 16)]
            out[name].append(Step(text, at, i, target))
    return out


def too_early(steps):
    """(product, reader, instructions between them) of every read in front of its time."""
    found = []
    for first in steps:
        if not first.product:
            continue
        need, ways, seen = WAIT[first.op], [(n, 0, frozenset(first.writes)) for n in first.next], {}
        while ways:
            i, waited, live = ways.pop()
            if i >= len(steps) or waited >= need or seen.get((i, live), need) <= waited:
                continue
            seen[i, live] = waited
            s = steps[i]
            if s.reads & live or (s.writes & live and not (s.product and s.adds & live)):
                found.append((first.text, s.text, waited))
                continue
            left = live - s.writes - s.adds
            if left:
                ways += [(n, waited + s.takes, left) for n in s.next]
    return found


def listing(body):
    lines = ["0000000000000100 <kernel>:"]
    at = 0x100
    for text in body:
        where = re.search(r"@(\d+)$", text)
        lines.append("\t%s // %012X: 00000000%s" % (text.split(" @")[0], at, " <kernel+0x%x>" % (4 * int(where[1])) if where else ""))
        at += 4
    return "\n".join(lines)


PRODUCT = "v_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], 0"
WAYS = {   # instructions (a branch's target behind @), and whether a result is read too early
    "straight, too early": ([PRODUCT, "s_nop 6", "v_mov_b32 v0, v7", "s_endpgm"], True),
    "straight": ([PRODUCT, "s_nop 7", "v_mov_b32 v0, v7", "s_endpgm"], False),
    "the way over a branch": ([PRODUCT, "s_cbranch_vccnz 1 @4", "s_nop 7", "s_nop 0", "ds_write_b32 v0, v6", "s_endpgm"], True),
    "the way over a branch, with its wait": ([PRODUCT, "s_cbranch_vccnz 1 @3", "s_nop 7", "s_nop 6", "ds_write_b32 v0, v6", "s_endpgm"], False),
    "round a loop": (["v_add_f32 v1, v5, v1", "s_nop 7", PRODUCT, "s_branch 0 @0"], True),
    "sums of sums": ([PRODUCT, "v_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], v[4:7]", "s_nop 7", "v_mov_b32 v0, v4", "s_endpgm"], False),
    "an operand": ([PRODUCT, "v_mfma_f32_16x16x32_bf16 v[16:19], v[4:7], v[12:15], 0", "s_endpgm"], True),
    "written over": ([PRODUCT, "v_mov_b32 v6, 0", "s_endpgm"], True),
}


@pytest.mark.parametrize("body,early", WAYS.values(), ids=WAYS.keys())
def test_the_check_itself(body, early):
    assert bool(too_early(parse(listing(body))["kernel"])) == early


def test_kernels_of_the_delta_rule(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no %s here" % OBJDUMP)
    with open(capi.HIP_LIB, "rb") as f:
        data = f.read()
    checked, at = 0, data.find(MAGIC)
    while at >= 0:
        entry = at + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", data, at + len(MAGIC))[0]):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            code = data[at + offset:at + offset + size]
            if b"gfx950" not in target or b"k_delta_chunks" not in code:
                continue
            (tmp_path / "code.co").write_bytes(code)
            text = subprocess.check_output([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", str(tmp_path / "code.co")], text=True)
            for name, steps in parse(text).items():
                if any(s.product for s in steps):
                    assert not too_early(steps), name
                    checked += 1
        at = data.find(MAGIC, at + 1)
    assert checked >= 40   # chunks and their preparation, six widths in two types; joins
