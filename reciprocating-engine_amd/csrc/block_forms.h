// block_forms.h - which kernel and tile the block-scaled fp8 product
// (csrc/gemm_blocks.hip) runs on. Plain C++ so that the host tests can check the
// choice with the code the launcher runs.
#pragma once

#include <stdint.h>

namespace reng {

enum BlockForm {
    BLK_RING_1x1,   // gemm_blocks_ring: 16 MT rows of a by 16 NT of b, the waves split k
    BLK_RING_1x4,
    BLK_RING_2x1,
    BLK_RING_2x2,
    BLK_RING_4x1,
    BLK_RING_4x2,
    BLK_RING_4x4,
    BLK_TILE_64,    // gemm_blocks_tiles
    BLK_TILE_128,
    BLK_TILE_256,
    BLK_FORMS,
};

// Outputs of a workgroup, blocks of k it takes a step, workgroups on a CU; the start of
// a round and a step's time (us) where there is a workgroup a CU at most, and where the
// CUs hold all they can. Fitted to graph-replayed timings of every form on 26 products
// (M 1 to 4096, N 1024 to 27648, K 512 to 18944); on these the choice is the fastest one
// or within 10% of it.
struct BlockCost {
    uint32_t bm, bn, step, per_cu;
    float start, one, all;
};
constexpr BlockCost BLOCK_COST[BLK_FORMS] = {
    {16, 16, 4, 2, 2.2f, 0.35f, 0.58f}, {16, 64, 4, 1, 2.2f, 1.35f, 1.35f}, {32, 16, 4, 1, 2.2f, 0.49f, 0.60f},
    {32, 32, 4, 2, 2.2f, 0.65f, 0.95f}, {64, 16, 4, 1, 2.2f, 0.80f, 0.95f}, {64, 32, 4, 1, 2.2f, 0.97f, 1.00f},
    {64, 64, 4, 1, 2.2f, 1.45f, 1.57f}, {64, 64, 1, 3, 2.5f, 0.43f, 0.70f}, {128, 128, 1, 2, 3.0f, 0.84f, 1.12f},
    {256, 256, 1, 1, 6.0f, 1.60f, 1.60f},
};

inline float block_cost(int form, uint64_t M, uint64_t N, uint64_t K, uint64_t cus) {
    const BlockCost &c = BLOCK_COST[form];
    const uint64_t wgs = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const uint64_t steps = ((K + 127) / 128 + c.step - 1) / c.step;
    if (wgs <= cus) return c.start + c.one * (float)steps;
    return (float)((wgs + cus * c.per_cu - 1) / (cus * c.per_cu)) * (c.start + c.all * (float)steps);
}

inline BlockForm block_pick(uint64_t M, uint64_t N, uint64_t K, uint64_t cus) {
    int best = BLK_RING_1x1;
    float us = -1.0f;
    for (int f = 0; f < BLK_FORMS; ++f) {
        // A form is for rows of a that its tile holds most of; the ring forms of 64 rows take any number.
        if (M <= 16 ? BLOCK_COST[f].bm > 16 : f < BLK_RING_2x1) continue;
        if (M > 32 && f < BLK_RING_4x1) continue;
        const float t = block_cost(f, M, N, K, cus);
        if (us < 0.0f || t < us) us = t, best = f;
    }
    return (BlockForm)best;
}

}  // namespace reng
