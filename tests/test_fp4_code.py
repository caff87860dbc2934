"""The built code of the 4-bit weights and caches: a matrix product's result is there 8
instructions (16 x 16 x 32) or 12 (32 x 32 x 16) after the product.  The compiler keeps
that in straight code; behind a branch it has read a score after 3, the score before
then.  All paths through each kernel are followed here."""
import os
import re
import subprocess

import pytest

from test_batch_code import OBJDUMP, code_object
from test_code_placement import LIB

REGISTER = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")
NEEDED = {"16x16x32": 8, "32x32x16": 12}


def registers(operand):
    return {(m[1], r) for m in REGISTER.finditer(operand) for r in range(int(m[2] or m[4]), int(m[3] or m[4]) + 1)}


class Step:
    def __init__(self, line):
        code, _, comment = line.partition("//")
        self.text = code.strip()
        self.address = int(comment.split(":")[0], 16)
        op, _, rest = self.text.partition(" ")
        operands = [x.strip() for x in rest.split(",")]
        self.states = int(rest, 0) + 1 if op == "s_nop" else 1
        self.needed = next((n for size, n in NEEDED.items() if op.startswith("v_mfma") and size in op), 0)
        self.target, self.ends = None, op in ("s_endpgm", "s_branch")
        self.written, self.read = set(), set()
        if op.startswith(("s_cbranch", "s_branch")):
            offset = int(operands[0], 0)
            self.target = self.address + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)
        elif self.needed:  # a product may follow the one whose sum it goes on with
            self.written, self.read = registers(operands[0]), registers(operands[1]) | registers(operands[2])
        elif op.startswith("v_"):
            self.written = registers(operands[0])
            swapped = operands if "swap" in op else operands[1:]
            self.read = set().union(*map(registers, swapped)) if swapped else set()
        elif op.startswith(("ds_", "global_", "buffer_", "flat_", "scratch_")):
            from_here = operands if "store" in op or "write" in op else operands[1:]
            self.read = set().union(*map(registers, from_here)) if from_here else set()


def early_reads(lines):
    """Instructions that read a product's result too soon on some path, and the products."""
    steps = [Step(line) for line in lines if "//" in line]
    place = {s.address: n for n, s in enumerate(steps)}
    joins = {place[s.target] for s in steps if s.target is not None}
    found, seen, paths = {}, {}, [(0, {})]
    while paths:
        n, left = paths.pop()
        left = dict(left)  # register: instructions still to wait
        while n < len(steps):
            s = steps[n]
            if n in joins:
                old = seen.get(n)
                if old is not None and all(old.get(r, 0) >= w for r, w in left.items()):
                    break
                left = {r: max(left.get(r, 0), (old or {}).get(r, 0)) for r in left.keys() | (old or {}).keys()}
                seen[n] = dict(left)
            for r in s.read & left.keys():
                found[n] = f"{s.text}: {left[r]} too soon"
            if not s.needed:
                for r in s.written:
                    left.pop(r, None)
            left = {r: w - s.states for r, w in left.items() if w > s.states}
            for r in s.written if s.needed else ():
                left[r] = s.needed
            if s.target is not None:
                paths.append((place[s.target], left))
            if s.ends:
                break
            n += 1
    return [found[n] for n in sorted(found)], sum(bool(s.needed) for s in steps)


FAULTY = """
  v_mfma_f32_16x16x32_bf16 a[20:23], v[0:3], v[4:7], a[20:23] // 0000: 0
  s_cbranch_vccnz 2 // 0008: 0
  s_nop 7 // 000C: 0
  s_branch 1 // 0010: 0
  s_nop 3 // 0014: 0
  v_accvgpr_read_b32 v55, a23 // 0018: 0
  s_endpgm // 0020: 0
"""


def test_the_check_sees_the_fault():
    assert early_reads(FAULTY.splitlines()) == (["v_accvgpr_read_b32 v55, a23: 3 too soon"], 1)
    assert early_reads(FAULTY.replace("s_nop 3", "s_nop 6").splitlines()) == ([], 1)


def test_products_are_read_when_they_are_there(tmp_path):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("libdlhip.so or the disassembler is not here")
    kernels = {}
    for kernel in (b"8k_attendI", b"14k_project_many"):
        image = code_object(LIB, b"3fp412_GLOBAL__N_1" + kernel)
        assert image is not None
        path = tmp_path / "fp4.co"
        path.write_bytes(image)
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True,
                                 check=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]+ <_ZN)", listing):
            name, _, body = part.partition("\n")
            if "3fp412" in name:
                kernels[name] = early_reads(body.splitlines())
    assert not {name: found[:3] for name, (found, _) in kernels.items() if found}
    for kernel in ("8k_attend", "16k_project_staged", "14k_project_many", "14k_project_long"):
        assert sum(count for name, (_, count) in kernels.items() if kernel in name) >= 16, kernel
