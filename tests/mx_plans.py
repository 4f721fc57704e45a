"""The choices of the 4-bit operators' launchers, from the headers that the launchers themselves use."""
import ctypes
import os
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reciprocating-engine_amd", "csrc")
CUS = 256   # an MI355X
SOURCE = """
#include "head_forms.h"
#include "mx_attention_plan.h"
#include "mx_forms.h"
using namespace reng;
extern "C" void plan(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, size_t cus, uint64_t *out) {
    const MxAttnPlan p = mxa_plan(nh, nkv, hd, len, tokens, cus);
    const uint64_t v[] = {p.hdp, (uint64_t)p.form, p.row_blocks, p.splits, p.tiles, mxa_part_bytes(p, nkv, tokens * (nh / nkv))};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
}
extern "C" int pick(uint64_t M, uint64_t N, uint64_t K, uint64_t cus) { return mx_pick(M, N, K, cus); }
extern "C" uint32_t row_waves(uint64_t N, uint64_t K, uint64_t cus) { return mx_row_waves(N, K, cus); }
extern "C" int by_four(uint64_t tokens, uint32_t heads, uint32_t group, int rotates, int mixed, uint64_t cus) {
    return heads_by_four(tokens, heads, group, rotates, mixed, cus);
}
extern "C" int forms() { return MX_FORMS; }
extern "C" void outputs(int form, uint32_t *out) { out[0] = MX_COST[form].bm, out[1] = MX_COST[form].bn; }
extern "C" void shape(uint32_t hdp, int form, uint32_t *out) {
    out[0] = mxa_shape(hdp, form).rows, out[1] = mxa_shape(hdp, form).tile;
}
"""
_lib = None


def lib():
    global _lib
    if _lib is None:
        with tempfile.TemporaryDirectory() as d:
            src, so = os.path.join(d, "plans.cpp"), os.path.join(d, "plans.so")
            with open(src, "w") as f:
                f.write(SOURCE)
            subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-o", so, src],
                           check=True)
            _lib = ctypes.CDLL(so)
        _lib.plan.argtypes = [ctypes.c_size_t] * 6 + [ctypes.c_void_p]
        _lib.pick.argtypes = [ctypes.c_uint64] * 4
        _lib.by_four.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int, ctypes.c_int, ctypes.c_uint64]
        _lib.row_waves.argtypes = [ctypes.c_uint64] * 3
    return _lib


def mx_attention_plan(nh, nkv, hd, length, tokens, cus=CUS):
    out = (ctypes.c_uint64 * 6)()
    lib().plan(nh, nkv, hd, length, tokens, cus, out)
    return dict(zip(("hdp", "form", "row_blocks", "splits", "tiles", "bytes"), out))


def shape(hdp, form):
    """Query rows of a workgroup and cache rows of a tile."""
    out = (ctypes.c_uint32 * 2)()
    lib().shape(hdp, form, out)
    return tuple(out)


def mx_form(M, N, K, cus=CUS):
    """The product's form for more than one row, and the outputs of one of its workgroups."""
    out = (ctypes.c_uint32 * 2)()
    form = lib().pick(M, N, K, cus)
    lib().outputs(form, out)
    return form, tuple(out)


def mx_forms():
    return lib().forms()


def mx_row_waves(N, K, cus=CUS):
    """The waves that share an output's k where a has one row."""
    return lib().row_waves(N, K, cus)


def head_lanes(hd):
    """Lanes of a head, eight values each."""
    return next(n // 8 for n in (32, 64, 128, 256) if hd <= n)


def heads_by_four(tokens, heads, hd, rotates=True, mixed=False, cus=CUS):
    """Whether a group of lanes takes four of a token's heads (queries, keys and values)."""
    return bool(lib().by_four(tokens, heads, 256 // head_lanes(hd), rotates, mixed, cus))


# (heads, kv, hd, length, tokens): with the attention tests' other cases every kernel, with and without a merge.
ATTENTION_SHAPES = [
    (8, 1, 32, 0, 65), (4, 1, 32, 910, 140), (7, 1, 32, 6262, 77), (5, 1, 64, 120, 436), (4, 1, 32, 162, 563),
    (4, 1, 32, 8227, 275), (16, 2, 64, 0, 556), (5, 1, 64, 0, 989), (7, 1, 32, 14568, 343), (15, 3, 96, 21, 214),
    (10, 2, 96, 1128, 279), (4, 1, 96, 4516, 148), (7, 1, 96, 2, 423), (4, 1, 96, 151, 942), (7, 1, 96, 6373, 151),
    (14, 2, 96, 45, 814), (16, 2, 128, 0, 542), (8, 1, 96, 39, 518), (5, 1, 128, 6331, 429), (21, 3, 160, 4, 106),
    (15, 3, 160, 646, 117), (5, 1, 160, 3007, 104), (8, 1, 160, 28, 264), (7, 1, 160, 28, 340), (5, 1, 256, 172, 690),
    (7, 1, 224, 5576, 153),
]
# (M, N, K): every form of the product, with edges inside tiles and stages.
PRODUCT_SHAPES = [
    (9, 33, 64), (2, 4169, 32), (2, 4435, 2240), (21, 2147, 1088), (17, 2058, 32), (4131, 21, 2016), (4255, 36, 32),
    (2185, 102, 2016), (39, 5111, 288), (41, 4469, 2432), (33, 8307, 928), (46, 9844, 2048), (33, 4584, 32), (42, 9667, 2144),
    (67, 8538, 32), (138, 11009, 2112), (1451, 8248, 1312), (2323, 5357, 1344),
]
# (N, K) of products of one row: one, two and four waves an output, even and odd N, whole and cut pieces of k.
ROW_SHAPES = [
    (1, 32), (7, 96), (129, 2048), (8193, 2080), (8194, 2080), (8192, 8192), (9001, 14336), (33, 4096), (1022, 6144), (4099, 8192),
    (4098, 8224), (4095, 6176), (1, 8192), (62, 9248), (7, 18944), (1021, 8224), (2048, 10240), (2049, 14336),
]
