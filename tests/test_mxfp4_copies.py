"""The copies into LDS of the MXFP4 product, in the code that hipcc makes of them for gfx950, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from test_lds_copies import LIB, OBJDUMP, Code, sgprs


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs llvm-objdump")
def test_no_copy_reads_a_resource_that_the_vector_unit_has_just_written(tmp_path):
    """Five wait states lie between the vector unit's write of a scalar register and a copy that reads it."""
    if not os.path.exists(LIB):
        pytest.skip("needs the built library")
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    copies = kernels = 0
    for f in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", f.name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            if not re.search(r"gemm_mx_(ring|tiles)", part.split("\n", 1)[0]):
                continue
            code, kernels = Code(part.splitlines()), kernels + 1
            for i, (name, ops, _) in enumerate(code.ins):
                if name == "buffer_load_dwordx4" and ops[-1].endswith("lds"):
                    copies += 1
                    regs = set().union(*(sgprs(o.split()[0]) for o in ops))
                    assert not code.valu_write_within(i, regs, 5), (part.split("\n", 1)[0], name, ops)
    assert kernels == 10 and copies >= 200, (kernels, copies)
