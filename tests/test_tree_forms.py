"""The tree attention's kernels and the shapes that the GPU tests reach them at:
the launcher's own choice (csrc/tree_plan.h), built on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "reciprocating-engine_amd", "csrc")
CUS = 256

# (head size the kernel is built for, its form, the merge's waves a row): heads, key/value heads, head size, context, tokens.
# Contexts that end inside a tile behind several steps of whole ones, and rows that leave the last row block short.
TREE_FORM_SHAPES = {
    (64, 0, 4): (4, 1, 56, 14889, 6), (64, 1, 0): (12, 6, 56, 601, 46), (64, 1, 1): (4, 1, 56, 2830, 259),
    (64, 1, 4): (28, 7, 64, 6547, 17), (64, 2, 0): (7, 1, 64, 195, 294), (64, 2, 1): (8, 1, 64, 971, 285),
    (64, 2, 4): (8, 1, 56, 1709, 261), (64, 3, 0): (8, 1, 64, 200, 526), (64, 3, 1): (8, 1, 64, 599, 538),
    (64, 3, 4): (3, 1, 56, 2408, 731),
    (96, 0, 4): (1, 1, 96, 17355, 12), (96, 1, 0): (16, 8, 96, 349, 34), (96, 1, 1): (24, 8, 88, 1868, 65),
    (96, 1, 4): (48, 8, 88, 5473, 11), (96, 2, 0): (8, 1, 88, 193, 289), (96, 2, 1): (8, 1, 96, 978, 265),
    (96, 2, 4): (7, 1, 88, 1657, 304), (96, 3, 0): (16, 2, 96, 213, 530), (96, 3, 1): (8, 1, 96, 600, 545),
    (96, 3, 4): (5, 1, 88, 3674, 460),
    (128, 0, 4): (3, 1, 128, 13024, 4), (128, 1, 0): (6, 2, 128, 315, 68), (128, 1, 1): (42, 6, 128, 1893, 37),
    (128, 1, 4): (36, 6, 112, 6567, 11), (128, 2, 0): (7, 1, 128, 193, 293), (128, 2, 1): (7, 1, 128, 982, 294),
    (128, 2, 4): (7, 1, 112, 1652, 308), (128, 3, 0): (16, 2, 128, 195, 527), (128, 3, 1): (8, 1, 128, 594, 542),
    (128, 3, 4): (8, 1, 112, 6920, 258),
    (256, 0, 0): (10, 5, 136, 274, 46), (256, 0, 1): (21, 7, 256, 942, 33), (256, 0, 4): (8, 2, 136, 18402, 1),
    (256, 1, 0): (7, 1, 256, 246, 159), (256, 1, 1): (7, 1, 256, 816, 172), (256, 1, 4): (4, 1, 136, 2049, 145),
    (256, 2, 0): (16, 2, 256, 102, 259), (256, 2, 1): (8, 1, 256, 389, 275), (256, 2, 4): (6, 1, 256, 1674, 363),
}

# The eight-wave form where it begins or ends at a border: no context, less than a tile, a tile, one row more.
TREE_EDGE_SHAPES = [(hd, 3, *s) for hd in (64, 96, 128)
                    for s in [(16, 2, hd, 0, 700), (16, 2, hd, 5, 700), (16, 2, hd, 63, 700), (16, 2, hd, 64, 700),
                              (16, 2, hd, 65, 700), (16, 2, hd, 640, 1024)]]

SOURCE = r"""
#include "tree_plan.h"
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>
using namespace reng;
int main(int argc, char **argv) {
    const size_t cus = atoi(argv[1]);
    if (argc == 2) {   // every kernel that a plan can name
        bool seen[4][4][5] = {};
        for (size_t hd : {(size_t)64, (size_t)96, (size_t)128, (size_t)256})
            for (size_t nkv = 1; nkv <= 16; nkv = nkv < 8 ? nkv + 1 : nkv * 2)
                for (size_t per : {(size_t)1, (size_t)4, (size_t)5, (size_t)7, (size_t)8})
                    for (size_t t = 1; t <= 1024; t = t * 5 / 4 + 1)
                        for (size_t len = 0; len < 100000; len = len * 5 / 4 + 7) {
                            const TreePlan p = tree_plan(nkv * per, nkv, hd, len, t, true, cus);
                            seen[hd == 64 ? 0 : hd == 96 ? 1 : hd == 128 ? 2 : 3][p.form][tree_merge_waves(p, nkv)] = true;
                        }
        const int sizes[4] = {64, 96, 128, 256};
        for (int h = 0; h < 4; ++h)
            for (int f = 0; f < 4; ++f)
                for (int m = 0; m < 5; ++m)
                    if (seen[h][f][m]) printf("%d %d %d\n", sizes[h], f, m);
        return 0;
    }
    for (int i = 2; i + 4 < argc; i += 5) {
        auto at = [&](int k) { return (size_t)strtoull(argv[i + k], 0, 10); };
        const TreePlan p = tree_plan(at(0), at(1), at(2), at(3), at(4), true, cus);
        printf("%u %d %u\n", p.hdp, p.form, tree_merge_waves(p, at(1)));
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("tree_forms")
    src, exe = d / "plans.cpp", d / "plans"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-o", str(exe), str(src)], check=True)

    def run(*shapes):
        out = subprocess.run([str(exe), str(CUS), *(str(v) for s in shapes for v in s)], check=True, capture_output=True,
                             text=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


def test_the_shapes_run_the_kernels_they_name(plans):
    assert plans(*TREE_FORM_SHAPES.values()) == list(TREE_FORM_SHAPES)
    assert [p[:2] for p in plans(*(s[2:] for s in TREE_EDGE_SHAPES))] == [s[:2] for s in TREE_EDGE_SHAPES]


def test_every_kernel_has_its_shapes(plans):
    """Form 0 without many splits is for caches of a few tiles (the smallest shapes of test_gpu_attention_tree.py)."""
    missing = {p for p in plans() if p not in TREE_FORM_SHAPES}
    assert missing <= {(hd, 0, m) for hd in (64, 96, 128) for m in (0, 1)}, missing
