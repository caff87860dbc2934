"""The built code of the batch attention: matrix operands are assembled from
loaded words by byte permutes.  With the next step's loads under a condition
the compiler has built an operand in the registers of a loaded row whose other
words were still to be read (a permute then took a permute's result for a
loaded word).  A permute here reads loaded words only, so that shows in the
listing."""
import os
import re
import struct
import subprocess

import pytest

from test_code_placement import EM_AMDGPU, LIB

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def code_object(path, kernel):
    """The bytes of the gfx950 image that holds the kernel."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(b"\x7fELF", 1)
    while at >= 0:
        end = data.find(b"\x7fELF", at + 1)
        image = data[at:end if end > 0 else None]
        if struct.unpack_from("<H", image, 18)[0] == EM_AMDGPU and kernel in image:
            return image
        at = end
    return None


def permutes_of_permutes(lines):
    """Permutes that read what an earlier permute of the same straight run of code wrote."""
    by_permute, found, count = set(), [], 0
    for line in lines:
        code = line.split("//")[0].split(";")[0].strip()
        if not code or code.endswith(":") or code.startswith(("s_cbranch", "s_branch", "s_setpc", "s_endpgm")):
            by_permute = set()
            continue
        op, _, operands = code.partition(" ")
        operands = [x.strip() for x in operands.split(",")]
        if op == "v_perm_b32":
            count += 1
            if by_permute & set(operands[1:3]):
                found.append(code)
            by_permute.add(operands[0])
        else:  # whatever else is written holds no permute's result
            written = re.fullmatch(r"v\[(\d+):(\d+)\]|v(\d+)", operands[0])
            if written:
                first, last = (written[1], written[2]) if written[1] else (written[3], written[3])
                by_permute -= {f"v{r}" for r in range(int(first), int(last) + 1)}
    return found, count


FAULTY = """
  v_perm_b32 v82, v86, v82, s86
  v_perm_b32 v83, v94, v90, s86
  v_mfma_f32_16x16x32_bf16 v[30:33], v[82:85], v[120:123], v[30:33]
  v_perm_b32 v82, v87, v83, s88
"""


def test_the_check_sees_the_fault():
    assert permutes_of_permutes(FAULTY.splitlines()) == (["v_perm_b32 v82, v87, v83, s88"], 3)
    loaded = FAULTY.replace("v_mfma", "global_load_dwordx4 v[82:85], v[2:3], off\n  v_mfma")
    assert permutes_of_permutes(loaded.splitlines()) == ([], 3)


def test_operands_are_assembled_from_loaded_words(tmp_path):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("libdlhip.so or the disassembler is not here")
    image = code_object(LIB, b"k_weights")
    assert image is not None
    path = tmp_path / "batch.co"
    path.write_bytes(image)
    listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], capture_output=True,
                             text=True, check=True).stdout
    total = 0
    for part in re.split(r"\n(?=<?\w*_ZN)", listing):
        name, _, body = part.partition("\n")
        if "8k_ranges" not in name:
            continue
        found, count = permutes_of_permutes(body.splitlines())
        assert not found, (name, found[:3])
        total += count
    assert total > 500  # every few-row BF16 form has at least 2 D / 8
