// mx_attention_plan.h - how the attention over a 4-bit cache (csrc/attention_mxfp4.hip)
// cuts its query rows into row blocks and its cache into splits. Plain C++ so that the
// host tests can check the plans with the code the launcher runs.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace reng {

constexpr uint32_t MXA_XCDS = 8, MXA_TILE = 32, MXA_SPLIT_MAX = 64;

// Eight waves with the same 16 query rows that take tiles of the cache in turn (four of 256
// dimensions); or workgroups of 64, 128 or 256 query rows that share tiles in LDS.
enum MxAttnForm { MXA_ROWS_16, MXA_TILES_64, MXA_TILES_128, MXA_TILES_256, MXA_FORMS };

// Query rows of a workgroup, cache rows of a tile and how many tiles it takes at a time; the start of
// a round of workgroups, one a CU, and a step's time (us).
struct MxAttnShape {
    uint32_t rows, tile, groups;
    float start, step;
};
constexpr MxAttnShape MXA_SHAPES[3][MXA_FORMS] = {
    {{16, 32, 8, 2.0f, 0.70f}, {64, 32, 4, 2.5f, 0.95f}, {128, 32, 2, 3.5f, 0.80f}, {256, 64, 1, 6.5f, 1.10f}},
    {{16, 32, 8, 2.5f, 1.10f}, {64, 32, 4, 6.5f, 1.25f}, {128, 32, 2, 5.5f, 1.10f}, {256, 64, 1, 4.5f, 1.65f}},
    {{16, 32, 4, 5.0f, 1.20f}, {64, 32, 2, 8.5f, 1.75f}, {128, 32, 1, 8.5f, 1.50f}, {0, 0, 0, 0.0f, 0.0f}},
};
// The merge's launch, and its share of a megabyte of partials. Fitted with the shapes' times to graph replays of
// every form with up to 64 splits on 24 calls (64, 128 and 256 dimensions, 1 to 1024 tokens, 0 to
// 131071 rows); on these the choice is the fastest or within 5% of it (one: 8%).
constexpr float MXA_MERGE_US = 5.5f, MXA_MERGE_US_MB = 0.55f;

// Query rows that splits leave, at most (68 MB of 128 dimensions), and the cache rows of a split, at least.
constexpr size_t MXA_PART_ROWS = 1 << 17, MXA_SPLIT_ROWS = 128;

struct MxAttnPlan {
    uint32_t hdp;           // the head size the kernel is built for: 64, 128 or 256
    int form;
    uint32_t row_blocks;    // per key/value head
    uint32_t splits, tiles; // of the cache, and all its tiles
};

inline uint32_t mxa_head(size_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
inline const MxAttnShape &mxa_shape(uint32_t hdp, int form) { return MXA_SHAPES[hdp == 64 ? 0 : hdp == 128 ? 1 : 2][form]; }

inline size_t mxa_most_splits(size_t cache) {
    const size_t s = cache / MXA_SPLIT_ROWS;
    return s < 1 ? 1 : s > MXA_SPLIT_MAX ? MXA_SPLIT_MAX : s;
}

// The cheapest form and number of splits. Rounds go by XCD: the row blocks of a split and
// key/value head run on one, and those units go to the XCDs in turn.
inline MxAttnPlan mxa_plan(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, size_t cus) {
    MxAttnPlan p{};
    p.hdp = mxa_head(hd);
    const size_t rows = tokens * (nh / nkv), cache = len + tokens, most = mxa_most_splits(cache);
    const size_t xcd = cus < MXA_XCDS ? 1 : cus / MXA_XCDS;
    float best = 0.0f;
    for (int f = 0; f < MXA_FORMS; ++f) {
        const MxAttnShape &sh = mxa_shape(p.hdp, f);
        // A form may leave less than three quarters of its rows without a query.
        if (sh.rows == 0 || (f > 0 && sh.rows >= 4 * rows)) continue;
        const size_t blocks = (rows + sh.rows - 1) / sh.rows, tiles = (cache + sh.tile - 1) / sh.tile;
        for (size_t s = 1; s <= most && (s == 1 || s * nkv * rows <= MXA_PART_ROWS); ++s) {
            const size_t rounds = ((s * nkv + MXA_XCDS - 1) / MXA_XCDS * blocks + xcd - 1) / xcd;
            const size_t steps = ((tiles + s - 1) / s + sh.groups - 1) / sh.groups;
            float us = (float)rounds * (sh.start + sh.step * (float)steps);
            if (s > 1) us += MXA_MERGE_US + MXA_MERGE_US_MB * 4e-6f * (float)(s * nkv * rows * (p.hdp + 2));
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

// A split leaves for each query row its unnormalised outputs, its maximum and its sum.
inline size_t mxa_part_bytes(const MxAttnPlan &p, size_t nkv, size_t rows) {
    return p.splits < 2 ? 0 : (size_t)p.splits * nkv * rows * (p.hdp + 2) * sizeof(float);
}

// No less than mxa_part_bytes asks for over 1 .. tokens tokens and 0 .. len context rows.
inline size_t mxa_workspace(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens) {
    const size_t splits = mxa_most_splits(len + tokens);
    if (splits < 2) return 0;
    size_t rows = splits * nkv * tokens * (nh / nkv);
    if (rows > MXA_PART_ROWS) rows = MXA_PART_ROWS;
    return rows * (mxa_head(hd) + 2) * sizeof(float);
}

}  // namespace reng
