// mx_attention_plan.h - how the attention over a 4-bit cache (csrc/attention_mxfp4.hip)
// cuts its query rows into row blocks and its cache into splits. Plain C++ so that the
// host tests can check the plans with the code the launcher runs.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace reng {

constexpr uint32_t MXA_XCDS = 8, MXA_WAVES = 4, MXA_TILE = 32, MXA_SPLIT_MAX = 64;

// Workgroups of a split cache, at most: their partials are 64 rows of at most 256 values each.
constexpr size_t MXA_PART_UNITS = 1024;

struct MxAttnPlan {
    uint32_t hdp;           // the head size the kernel is built for: 64, 128 or 256
    uint32_t qt;            // 16-row query tiles of a wave
    uint32_t row_blocks;    // per key/value head
    uint32_t splits, tiles; // of the cache, and all its tiles
};

inline uint32_t mxa_head(size_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

// Query tiles of a wave: as many as its rows ask for, four at most (two of 256 dimensions).
inline uint32_t mxa_tiles(size_t rows, uint32_t hdp) {
    if (rows <= 16) return 1;
    return rows <= 32 || hdp == 256 ? 2 : 4;
}

inline MxAttnPlan mxa_plan(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, size_t cus) {
    MxAttnPlan p{};
    p.hdp = mxa_head(hd);
    const size_t rows = tokens * (nh / nkv), cache = len + tokens;
    p.qt = mxa_tiles(rows, p.hdp);
    const size_t blocks = (rows + 16 * p.qt - 1) / (16 * p.qt), tiles = (cache + MXA_TILE - 1) / MXA_TILE;
    p.row_blocks = (uint32_t)blocks;
    p.tiles = (uint32_t)tiles;
    // Two workgroups a CU, each wave with a tile or more.
    const size_t units = nkv * blocks, want = 2 * cus / units, most = tiles / MXA_WAVES;
    size_t s = want < most ? want : most;
    if (s > MXA_SPLIT_MAX) s = MXA_SPLIT_MAX;
    if (s * units > MXA_PART_UNITS) s = MXA_PART_UNITS / units;
    p.splits = (uint32_t)(s < 1 ? 1 : s);
    return p;
}

// A split leaves for each query row its unnormalised outputs, its maximum and its sum.
inline size_t mxa_part_bytes(const MxAttnPlan &p, size_t nkv, size_t rows) {
    return p.splits < 2 ? 0 : (size_t)p.splits * nkv * rows * (p.hdp + 2) * sizeof(float);
}

// No less than mxa_part_bytes asks for over 1 .. tokens tokens and 0 .. len context rows:
// splits are at most a tile a wave, and splits times row blocks at most MXA_PART_UNITS.
inline size_t mxa_workspace(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens) {
    const size_t tiles = (len + tokens + MXA_TILE - 1) / MXA_TILE;
    size_t splits = tiles / MXA_WAVES;
    if (splits > MXA_SPLIT_MAX) splits = MXA_SPLIT_MAX;
    if (splits < 2) return 0;
    const uint32_t hdp = mxa_head(hd);
    size_t rows = splits * nkv * tokens * (nh / nkv);
    const size_t most = MXA_PART_UNITS * 16 * (hdp == 256 ? 2 : 4);
    if (rows > most) rows = most;
    return rows * (hdp + 2) * sizeof(float);
}

}  // namespace reng
