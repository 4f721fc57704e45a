"""The inline-asm copies into LDS (csrc/mfma_pipe.h, copy16_buf_asm), checked in
the code that hipcc makes of them for gfx950, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "reciprocating-engine_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

MIXED = r"""
#include "mfma_pipe.h"
using namespace reng;
__global__ void mixed(const void *p, const void *q, float *out) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2048];
    auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, 4096, 0x00020000);
    auto s = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(q), 0, 4096, 0x00020000);
    pipe::copy16_buf(r, lds, threadIdx.x * 16, 0);
    pipe::copy16_buf_asm(s, lds + 1024, threadIdx.x * 16);
    pipe::copy16_buf(r, lds, threadIdx.x * 16, 1024);
    pipe::wait_vmcnt<0>();
    __syncthreads();
    out[threadIdx.x] = *(float *)(lds + threadIdx.x * 4) + *(float *)(lds + 1024 + threadIdx.x * 4);
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_a_copy_by_the_compiler_after_one_in_asm_has_its_own_address(tmp_path):
    """m0 holds a copy's LDS address: the compiler has to know that the asm changes it, or it keeps what it set itself."""
    src = tmp_path / "mixed.hip"
    src.write_text(MIXED)
    run = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Wall", "-Werror",
                          "-Wno-unused-command-line-argument", "-I", CSRC, "--cuda-device-only", "-S", str(src), "-o", "-"],
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    lines = [x.strip() for x in run.stdout.splitlines()]
    lines = [x for x in lines if re.match(r"s_mov_b32 m0,|buffer_load_dwordx4 .* lds", x)]
    # Each copy behind a write of m0 of its own; the first and the last to the same address.
    assert [x.split()[0] for x in lines] == ["s_mov_b32", "buffer_load_dwordx4"] * 3, lines
    assert lines[0] == lines[4] != lines[2], lines
