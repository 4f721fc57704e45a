// tree_plan.h - how the tree attention (csrc/attention_tree.hip) cuts its query
// rows into row blocks and its cache into splits. Plain C++ so that the host
// tests can check the plans with the code the launcher runs.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace reng {

constexpr uint32_t TREE_XCDS = 8, TREE_SPLIT_MAX = 64;

// A workgroup's waves: rw of them take 32 query rows each, kw such groups take
// tiles of tk cache rows in turn.
struct TreeForm {
    uint32_t rw, kw, tk;
};

struct TreePlan {
    bool fast;              // the tiled kernel; else the general one
    uint32_t hdp;           // the head size the tiled kernel is built for: 64, 96, 128 or 256
    int form;               // index into the forms of that head size
    uint32_t row_blocks;    // per key/value head
    uint32_t splits, tiles; // of the cache, and all its tiles
};

constexpr TreeForm TREE_FORMS[4] = {{1, 2, 32}, {2, 4, 32}, {4, 2, 32}, {8, 1, 64}};
constexpr TreeForm TREE_FORMS_256[3] = {{1, 2, 32}, {2, 2, 32}, {4, 1, 32}};

inline TreeForm tree_form(uint32_t hdp, int form) { return hdp == 256 ? TREE_FORMS_256[form] : TREE_FORMS[form]; }

// What a wave leaves of a split: for 32 rows the unnormalised outputs, as its 64 lanes hold
// them, and each lane's maximum and sum.
#if defined(__HIPCC__)
__host__ __device__
#endif
constexpr uint32_t tree_wave_floats(uint32_t hdp) { return hdp * 32 + 128; }

// At most 64 splits of 64 rows or more, and 4096 waves' partials (68 MB at 128 dimensions).
constexpr size_t TREE_SPLIT_ROWS = 64, TREE_PART_WAVES = 4096;

inline size_t tree_most_splits(size_t cache) {
    const size_t s = cache / TREE_SPLIT_ROWS;
    return s < 1 ? 1 : s > TREE_SPLIT_MAX ? TREE_SPLIT_MAX : s;
}

// What a choice weighs: a step's microseconds by form and head size, 64, 96, 128 and 256; the
// start of a round of workgroups, the merge's launch, and its share of a megabyte of partials.
// They put forms and splits in order and are below the times themselves (the eight-wave form's
// step takes about 2 us at 128 dimensions). Graph replays of every form with up to 64 splits:
// us by the model, as chosen (form, splits), and at best.
//   32 heads on 8 of 128, 16 tokens after 500    10   15.2 (1, 5)    12.6 (0, 8)
//   the same, one token after 4096               13   17.8 (0, 22)   15.8 (0, 32)
//   one token after 32768                        29   38.7 (0, 31)   36.3 (0, 32)
//   63 after 32768                               53   54.7 (3, 27)   53.2 (3, 26)
//   28 on 4 of 128, 255 after 8191               51   53.4 (3, 7)    52.5 (3, 8)
//   40 on 8 of 128, chain of 1024 after 0        25   48.1 (3, 1)    the same
//   the same after 16384                        294    357 (3, 3)    the same
//   28 on 4 of 64, 100 after 9000                24   25.6 (2, 10)   25.1 (1, 9)
//   32 on 8 of 96, chain of 300 after 4000       38   39.3 (3, 5)    37.6 (3, 6)
//   16 on 2 of 256, 27 after 30000               40   45.5 (1, 32)   41.7 (2, 64)
constexpr float TREE_STEP_US[4][4] = {
    {0.70f, 0.90f, 1.05f, 1.30f}, {0.80f, 1.10f, 1.40f, 1.35f}, {0.70f, 0.95f, 1.10f, 1.50f}, {0.80f, 1.10f, 1.30f, 0.0f}};
constexpr float TREE_ROUND_US = 4.0f, TREE_MERGE_US = 4.0f, TREE_MERGE_US_MB = 0.7f;

// The cheapest form and number of splits. Rounds go by XCD: the row blocks of a split and
// key/value head run on one, and those units go to the XCDs in turn. A form may leave less than
// half of its row blocks' rows without a query.
inline TreePlan tree_plan(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, bool aligned, size_t cus) {
    TreePlan p{};
    p.fast = hd % 8 == 0 && hd <= 256 && aligned;
    p.splits = 1;
    if (!p.fast) return p;
    p.hdp = hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256;
    const int col = p.hdp == 64 ? 0 : p.hdp == 96 ? 1 : p.hdp == 128 ? 2 : 3;
    const size_t cache = len + tokens, most = tree_most_splits(cache);
    const size_t tiles32 = (tokens * (nh / nkv) + 31) / 32;   // 32-row tiles of a key/value head
    const size_t xcd = cus < TREE_XCDS ? 1 : cus / TREE_XCDS;
    float best = 0.0f;
    for (int f = 0; f < (p.hdp == 256 ? 3 : 4); ++f) {
        const TreeForm form = tree_form(p.hdp, f);
        if (f > 0 && form.rw >= 2 * tiles32) break;
        const size_t blocks = (tiles32 + form.rw - 1) / form.rw, tiles = (cache + form.tk - 1) / form.tk;
        for (size_t s = 1; s <= most; ++s) {
            const size_t waves = s * nkv * blocks * form.rw;
            if (s > 1 && waves > TREE_PART_WAVES) break;
            const size_t rounds = ((s * nkv + TREE_XCDS - 1) / TREE_XCDS * blocks + xcd - 1) / xcd;
            const size_t steps = ((tiles + s - 1) / s + form.kw - 1) / form.kw;
            float us = (float)rounds * (TREE_ROUND_US + TREE_STEP_US[f][col] * (float)steps);
            if (s > 1) us += TREE_MERGE_US + TREE_MERGE_US_MB * 4e-6f * (float)(waves * tree_wave_floats(p.hdp));
            if (best == 0.0f || us < best) {
                best = us;
                p.form = f;
                p.row_blocks = (uint32_t)blocks;
                p.tiles = (uint32_t)tiles;
                p.splits = (uint32_t)s;
            }
        }
    }
    return p;
}

inline size_t tree_part_bytes(const TreePlan &p, size_t nkv) {
    return p.splits < 2 ? 0
                        : (size_t)p.splits * nkv * p.row_blocks * tree_form(p.hdp, p.form).rw *
                              tree_wave_floats(p.hdp) * sizeof(float);
}

// Waves of the merge that share a row's splits: a workgroup's four where it has few rows to
// merge (at most a few workgroups a CU) from many splits; 0: nothing to merge.
inline uint32_t tree_merge_waves(const TreePlan &p, size_t nkv) {
    if (p.splits < 2) return 0;
    return p.splits >= 8 && nkv * p.row_blocks * tree_form(p.hdp, p.form).rw * (p.hdp / 8) <= 4096 ? 4 : 1;
}

// No less than tree_part_bytes asks for over 1 .. tokens tokens and 0 .. len context rows.
inline size_t tree_workspace(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens) {
    const size_t most = tree_most_splits(len + tokens);
    if (hd % 8 || hd > 256 || most < 2) return 0;
    const size_t tiles32 = (tokens * (nh / nkv) + 31) / 32;
    size_t waves = most * nkv * 2 * tiles32;
    if (waves > TREE_PART_WAVES) waves = TREE_PART_WAVES;
    return waves * tree_wave_floats(hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256) * sizeof(float);
}

}  // namespace reng
