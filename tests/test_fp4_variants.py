"""The built kernels of the operations over 4-bit storage: none is another's copy under a
second name, as the projection's FP32 forms for rows in whole pieces once were."""
import os
import re
import subprocess

import pytest

from test_batch_code import OBJDUMP, code_object
from test_code_placement import LIB


@pytest.mark.parametrize("kernel", [b"14k_project_many", b"8k_attendI"])
def test_no_kernel_is_built_twice(tmp_path, kernel):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("libdlhip.so or the disassembler is not here")
    image = code_object(LIB, b"3fp412_GLOBAL__N_1" + kernel)
    assert image is not None
    path = tmp_path / "fp4.co"
    path.write_bytes(image)
    listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], capture_output=True,
                             text=True, check=True).stdout
    bodies = {}
    for part in re.split(r"\n(?=<?\w*_ZN)", listing):
        name, _, body = part.partition("\n")
        if "3fp412" in name:
            # operations without their registers and addresses, which two compilations of one source may differ in
            steps = [line.split("//")[0].split()[0] for line in body.splitlines() if line.split("//")[0].strip()]
            steps = sorted(x for x in steps if not x.startswith(("s_nop", "s_code_end", "s_waitcnt")))
            bodies.setdefault(tuple(steps), []).append(name.strip("<>:"))
    assert len(bodies) > 10
    assert not [names for names in bodies.values() if len(names) > 1]
