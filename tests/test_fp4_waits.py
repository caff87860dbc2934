"""The built code of the attention over 4-bit caches: its wavefronts join through LDS
rooms that loads past the last step are sent to.  Before a barrier of the join no such
load may be under way, on any path: one that lands later would overwrite an output."""
import os
import re
import subprocess

import pytest

from test_batch_code import OBJDUMP, code_object
from test_code_placement import LIB


def barriers_with_loads(lines):
    """Addresses of barriers that a path reaches with loads to LDS under way, and the number of barriers."""
    steps = []
    for line in lines:
        code, found, comment = line.partition("//")
        if found:
            steps.append((int(comment.split(":")[0], 16), *code.strip().partition(" ")[::2]))
    place = {address: n for n, (address, _, _) in enumerate(steps)}
    seen, early, paths = set(), set(), [(0, False)]
    while paths:
        n, under_way = paths.pop()
        while n < len(steps) and (n, under_way) not in seen:
            seen.add((n, under_way))
            address, op, rest = steps[n]
            if "load_lds" in op:
                under_way = True
            elif op == "s_waitcnt" and re.search(r"vmcnt\(0\)", rest):
                under_way = False
            elif op == "s_barrier" and under_way:
                early.add(hex(address))
            if op.startswith(("s_cbranch", "s_branch")):
                offset = int(rest.split(",")[0], 0)
                paths.append((place[address + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)], under_way))
            if op in ("s_endpgm", "s_branch"):
                break
            n += 1
    return sorted(early), sum(op == "s_barrier" for _, op, _ in steps)


LISTING = """
  global_load_lds_dwordx4 v[2:3], off // 0000: 0
  s_waitcnt vmcnt(8) // 0008: 0
  s_cbranch_scc1 65532 // 000C: 0
  s_waitcnt vmcnt(0) lgkmcnt(0) // 0010: 0
  s_barrier // 0014: 0
  s_endpgm // 0018: 0
"""


def test_the_check_sees_a_missing_wait():
    assert barriers_with_loads(LISTING.splitlines()) == ([], 1)
    assert barriers_with_loads(LISTING.replace("vmcnt(0)", "vmcnt(1)").splitlines()) == (["0x14"], 1)
    assert barriers_with_loads(LISTING.replace("65532", "1").splitlines()) == (["0x14"], 1)


def test_no_load_is_under_way_at_the_join(tmp_path):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("libdlhip.so or the disassembler is not here")
    image = code_object(LIB, b"3fp412_GLOBAL__N_18k_attendI")
    assert image is not None
    path = tmp_path / "fp4.co"
    path.write_bytes(image)
    listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True, check=True).stdout
    kernels = {}
    for part in re.split(r"\n(?=[0-9a-f]+ <_ZN)", listing):
        name, _, body = part.partition("\n")
        if "8k_attend" in name:
            kernels[name] = barriers_with_loads(body.splitlines())
    assert len(kernels) >= 21
    assert not {name: early for name, (early, _) in kernels.items() if early}
    assert all(count >= 4 for _, count in kernels.values())


def test_the_source_waits_before_the_join():
    """The compiler keeps its own wait before a barrier by its own account of loads; the kernel's does not hang on it."""
    with open(os.path.join(os.path.dirname(LIB), "csrc", "fp4_attention.hip")) as f:
        kernel = f.read().split("void k_attend(")[1].split("\n}\n")[0]
    after_steps = kernel.split("uint32_t step = begin + wave;")[1]
    assert "s_waitcnt(lds_wait(0))" in after_steps.split("__syncthreads()")[0]
