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


OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LIB = os.path.join(ROOT, "reciprocating-engine_amd", "lib", "libreng_hip.so")


def sgprs(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand) or re.fullmatch(r"s(\d+)()", operand)
    return set(range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1)) if m else set()


class Code:
    """The instructions of a disassembled function: (mnemonic, operands, target offset of a branch)."""

    def __init__(self, lines):
        self.ins, at, first = [], {}, None
        for line in lines:
            m = re.match(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):[^<]*(?:<.*\+0x([0-9a-f]+)>)?", line)
            if not m:
                continue
            first = int(m.group(3), 16) if first is None else first
            at[int(m.group(3), 16) - first] = len(self.ins)
            ops = [x.strip() for x in re.split(r",(?![^\[]*\])", m.group(2))]
            self.ins.append((m.group(1), ops, int(m.group(4), 16) if m.group(4) else None))
        self.sources = {}
        for i, (name, _, target) in enumerate(self.ins):
            if name.startswith(("s_cbranch", "s_branch")) and target in at:
                self.sources.setdefault(at[target], []).append(i)

    def before(self, i):
        if i and self.ins[i - 1][0] not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            yield i - 1
        yield from self.sources.get(i, ())

    def valu_write_within(self, i, regs, states):
        """An instruction on the vector unit that writes one of regs fewer than `states` wait states before instruction i."""
        for p in self.before(i):
            name, ops, _ = self.ins[p]
            if name.startswith("v_") and regs & set().union(*(sgprs(o) for o in ops[:2 if "_co_" in name or "div_scale" in name else 1])):
                return self.ins[p]
            left = states - (int(ops[0], 0) + 1 if name == "s_nop" else 1)
            if left > 0:
                bad = self.valu_write_within(p, regs, left)
                if bad:
                    return bad
        return None


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs llvm-objdump")
def test_no_copy_reads_a_resource_that_the_vector_unit_has_just_written(tmp_path):
    """A vector-memory instruction may read a scalar register only five wait states after the vector unit wrote it. The
    compiler sees to that, but not inside an asm, which has two of its own."""
    if not os.path.exists(LIB):
        pytest.skip("needs the built library")
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    copies = kernels = 0
    for f in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", f.name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            if not re.search(r"attention_tree_tiles|gemm_blocks_", part.split("\n", 1)[0]):
                continue
            code, kernels = Code(part.splitlines()), kernels + 1
            for i, (name, ops, _) in enumerate(code.ins):
                if name == "buffer_load_dwordx4" and ops[-1].endswith("lds"):
                    copies += 1
                    regs = set().union(*(sgprs(o.split()[0]) for o in ops))
                    assert not code.valu_write_within(i, regs, 5), (part.split("\n", 1)[0], name, ops)
    assert kernels >= 15 and copies >= 1000, (kernels, copies)


def test_the_scan_finds_such_a_write():
    """The scan over instructions by hand: straight, across a branch, and far enough away."""
    def found(*lines):
        text = [f"\t{x}    // {0x1000 + 4 * i:012X}: 00000000{b}" for i, (x, b) in
                enumerate((x, "") if isinstance(x, str) else x for x in lines)]
        code = Code(text)
        return bool(code.valu_write_within(len(code.ins) - 1, {8, 9, 10, 11}, 5))

    load = "buffer_load_dwordx4 v1, s[8:11], 0 offen lds"
    assert found("v_readlane_b32 s9, v2, 3", "s_mov_b32 m0, s2", "s_nop 0", load)
    assert found("v_cmp_eq_u32_e64 s[10:11], 0, v1", "s_nop 3", load)
    assert not found("v_cmp_eq_u32_e64 s[10:11], 0, v1", "s_nop 4", load)
    assert not found("v_readlane_b32 s12, v2, 3", "s_nop 0", load)
    assert found("v_readfirstlane_b32 s8, v2", ("s_branch 2", " <f+0x10>"), "s_nop 4", "s_endpgm", load)
