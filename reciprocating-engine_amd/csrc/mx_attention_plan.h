// mx_attention_plan.h - how the attention over a 4-bit cache (csrc/attention_mxfp4.hip)
// cuts its query rows into row blocks and its cache into splits. Plain C++ so that the
// host tests can check the plans with the code the launcher runs.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace reng {

constexpr uint32_t MXA_XCDS = 8, MXA_WAVES = 4, MXA_TILE = 32, MXA_SPLIT_MAX = 64;

// Waves with query rows of their own (16, 32 or 64), four of which share a split's tiles; or
// workgroups of 64, 128 or 256 query rows that share tiles in LDS.
enum MxAttnForm { MXA_ROWS_16, MXA_ROWS_32, MXA_ROWS_64, MXA_TILES_64, MXA_TILES_128, MXA_TILES_256, MXA_FORMS };

// Query rows of a workgroup, cache rows of a tile, and how many tiles it takes at a time.
struct MxAttnShape {
    uint32_t rows, tile, groups;
};
constexpr MxAttnShape MXA_SHAPES[MXA_FORMS] = {{16, 32, 4}, {32, 32, 4}, {64, 32, 4}, {64, 32, 4}, {128, 32, 2}, {256, 64, 1}};
constexpr MxAttnShape MXA_SHAPES_256[MXA_FORMS] = {{16, 32, 4}, {32, 32, 4}, {0, 0, 0}, {64, 32, 2}, {128, 32, 1}, {0, 0, 0}};

inline MxAttnShape mxa_shape(uint32_t hdp, int form) { return hdp == 256 ? MXA_SHAPES_256[form] : MXA_SHAPES[form]; }

// Query rows that splits leave, at most (68 MB of 128 dimensions).
constexpr size_t MXA_PART_ROWS = 1 << 17;

struct MxAttnPlan {
    uint32_t hdp;           // the head size the kernel is built for: 64, 128 or 256
    int form;
    uint32_t row_blocks;    // per key/value head
    uint32_t splits, tiles; // of the cache, and all its tiles
};

inline uint32_t mxa_head(size_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

inline int mxa_form(size_t rows, uint32_t hdp) {
    if (rows <= 16) return MXA_ROWS_16;
    if (rows <= 32) return MXA_ROWS_32;
    if (rows <= 64) return MXA_TILES_64;
    return rows <= 128 || hdp == 256 ? MXA_TILES_128 : MXA_TILES_256;
}

inline MxAttnPlan mxa_plan_of(int form, size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, size_t cus) {
    MxAttnPlan p{};
    p.hdp = mxa_head(hd);
    const size_t rows = tokens * (nh / nkv), cache = len + tokens;
    p.form = form;
    const MxAttnShape s = mxa_shape(p.hdp, form);
    const size_t blocks = (rows + s.rows - 1) / s.rows, tiles = (cache + s.tile - 1) / s.tile;
    p.row_blocks = (uint32_t)blocks;
    p.tiles = (uint32_t)tiles;
    // Two workgroups of four waves a CU, or one of eight, and every group of waves with a tile or more.
    const size_t units = nkv * blocks, want = (form <= MXA_ROWS_64 ? 2 : 1) * cus / units, most = cache / 128;
    size_t n = want < most ? want : most;
    if (n > MXA_SPLIT_MAX) n = MXA_SPLIT_MAX;
    if (n > tiles) n = tiles;
    if (n * nkv * rows > MXA_PART_ROWS) n = MXA_PART_ROWS / (nkv * rows);
    p.splits = (uint32_t)(n < 1 ? 1 : n);
    return p;
}

inline MxAttnPlan mxa_plan(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, size_t cus) {
    return mxa_plan_of(mxa_form(tokens * (nh / nkv), mxa_head(hd)), nh, nkv, hd, len, tokens, cus);
}

// A split leaves for each query row its unnormalised outputs, its maximum and its sum.
inline size_t mxa_part_bytes(const MxAttnPlan &p, size_t nkv, size_t rows) {
    return p.splits < 2 ? 0 : (size_t)p.splits * nkv * rows * (p.hdp + 2) * sizeof(float);
}

// No less than mxa_part_bytes asks for over 1 .. tokens tokens and 0 .. len context rows:
// splits are of 128 cache rows or more, and splits times query rows at most 2^17.
inline size_t mxa_workspace(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens) {
    size_t splits = (len + tokens) / 128;
    if (splits > MXA_SPLIT_MAX) splits = MXA_SPLIT_MAX;
    if (splits < 2) return 0;
    size_t rows = splits * nkv * tokens * (nh / nkv);
    if (rows > MXA_PART_ROWS) rows = MXA_PART_ROWS;
    return rows * (mxa_head(hd) + 2) * sizeof(float);
}

}  // namespace reng
