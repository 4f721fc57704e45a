"""Which form a block-scaled product runs on and how the tree attention is cut:
the launchers' own code (csrc/block_forms.h, csrc/tree_plan.h), built on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "reciprocating-engine_amd", "csrc")
CUS = 256

# (form, M, N, K): the shapes the GPU tests run each form at.
FORM_SHAPES = [
    ("RING_1x1", 1, 4096, 640), ("RING_1x1", 13, 1000, 1168), ("RING_1x4", 1, 16400, 144), ("RING_1x4", 7, 14340, 528),
    ("RING_2x1", 17, 500, 1168), ("RING_2x1", 32, 1021, 512), ("RING_2x2", 20, 14002, 1040), ("RING_2x2", 31, 12001, 640),
    ("RING_4x1", 33, 1500, 2048), ("RING_4x1", 64, 1021, 1168), ("RING_4x2", 65, 2050, 1168), ("RING_4x2", 100, 4090, 2064), ("RING_4x4", 109, 5290, 7056),
    ("TILE_64", 64, 520, 16), ("TILE_64", 333, 1534, 576), ("TILE_64", 500, 2500, 1040),
    ("TILE_128", 700, 5001, 1168), ("TILE_128", 1100, 3300, 272), ("TILE_256", 2049, 4100, 1168),
    ("TILE_256", 4096, 4096, 144), ("TILE_256", 4001, 4090, 656), ("TILE_256", 3000, 5112, 512),
]

SOURCE = r"""
#include "block_forms.h"
#include "tree_plan.h"
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
using namespace reng;
int main(int argc, char **argv) {
    static const char *names[] = {"RING_1x1", "RING_1x4", "RING_2x1", "RING_2x2", "RING_4x1", "RING_4x2", "RING_4x4",
                                  "TILE_64", "TILE_128", "TILE_256"};
    const unsigned cus = atoi(argv[2]);
    if (!strcmp(argv[1], "form")) {
        for (int i = 3; i + 2 < argc; i += 3)
            puts(names[block_pick(strtoull(argv[i], 0, 10), strtoull(argv[i + 1], 0, 10), strtoull(argv[i + 2], 0, 10), cus)]);
        return 0;
    }
    if (!strcmp(argv[1], "sweep")) {   // every form the pick can give, over a grid of products
        bool seen[BLK_FORMS] = {};
        for (unsigned m = 1; m <= 4096; m = m * 3 / 2 + 1)
            for (unsigned n = 16; n <= 32768; n = n * 3 / 2 + 7)
                for (unsigned k = 128; k <= 32768; k *= 2) seen[block_pick(m, n, k, cus)] = true;
        for (int f = 0; f < BLK_FORMS; ++f)
            if (seen[f]) puts(names[f]);
        return 0;
    }
    // Tree plans: every query row in a block, every cache row in a tile, no empty split, the workspace large enough for
    // every smaller call.
    srand(7);
    for (int i = 0; i < 100000; ++i) {
        size_t nkv = 1 + rand() % 16, nh = nkv * (1 + rand() % 16), hd = 8 * (1 + rand() % 32), t = 1 + rand() % 1024;
        size_t len = rand() % (131072 - t);
        if (rand() % 2) len %= 2000;
        if (rand() % 2) t = 1 + t % 40;
        const size_t most = tree_workspace(nh, nkv, hd, len, t), t2 = 1 + rand() % t, l2 = rand() % (len + 1);
        const TreePlan p = tree_plan(nh, nkv, hd, l2, t2, true, cus);
        const TreeForm f = tree_form(p.hdp, p.form);
        if (!p.fast || p.hdp < hd || (size_t)p.row_blocks * f.rw * 32 < t2 * (nh / nkv) || p.splits > p.tiles ||
            (size_t)p.tiles * f.tk < l2 + t2 || tree_part_bytes(p, nkv) > most ||
            tree_workspace(nh, nkv, hd, l2, t2) > most) {
            printf("bad plan: %zu %zu %zu %zu %zu\n", nh, nkv, hd, l2, t2);
            return 1;
        }
    }
    if (tree_plan(8, 2, 80, 10, 1, false, cus).fast || tree_plan(8, 2, 82, 10, 1, true, cus).fast ||
        tree_plan(8, 2, 264, 10, 1, true, cus).fast)
        return 1;
    puts("ok");
    return 0;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("plans")
    src, exe = d / "plans.cpp", d / "plans"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-o", str(exe), str(src)], check=True)
    return lambda *a: subprocess.run([str(exe), *map(str, a)], check=True, capture_output=True, text=True).stdout.split()


def test_the_shapes_run_the_forms_they_name(plans):
    args = [v for s in FORM_SHAPES for v in s[1:]]
    assert plans("form", CUS, *args) == [s[0] for s in FORM_SHAPES]


def test_every_form_is_picked_somewhere(plans):
    seen = set(plans("sweep", CUS))
    assert seen == {s[0] for s in FORM_SHAPES}


@pytest.mark.parametrize("cus", [256, 64, 8, 1])
def test_tree_plans(plans, cus):
    assert plans("tree", cus) == ["ok"]
