// mx_forms.h - which kernel and tile the MXFP4 product (csrc/gemm_mxfp4.hip) runs
// on. Plain C++ so that the host tests can check the choice with the code the
// launcher runs.
#pragma once

#include <stdint.h>

namespace reng {

enum MxForm {
    MX_RING_1x1,   // gemm_mx_ring: 16 MT rows of a by 16 NT of b, the waves split k
    MX_RING_1x2,
    MX_RING_2x1,
    MX_RING_2x2,
    MX_RING_4x1,
    MX_RING_4x2,
    MX_RING_4x4,
    MX_TILE_64,    // gemm_mx_tiles
    MX_TILE_128,
    MX_TILE_256,
    MX_FORMS,
};

// Outputs of a workgroup, stages of 256 k it takes a step, workgroups that share a CU; the start of a
// round and a step's time (us) where there is a workgroup a CU at most, and where there are
// more. Fitted to graph-replayed timings of every form on 32 products (M 5 to 4096, N 1024 to
// 27648, K 576 to 27648); on these the choice is the fastest one or within 14% of it, but for
// 64 rows [3584, 18944] (27.2 us, and 19.6 on the 32 x 32 ring).
struct MxCost {
    uint32_t bm, bn, step, per_cu;
    float start, one, more;
};
constexpr MxCost MX_COST[MX_FORMS] = {
    {16, 16, 4, 3, 3.0f, 0.48f, 0.64f}, {16, 32, 4, 3, 3.0f, 0.64f, 1.22f}, {32, 16, 4, 2, 2.5f, 0.64f, 0.86f},
    {32, 32, 4, 3, 2.5f, 0.86f, 1.30f}, {64, 16, 4, 1, 2.0f, 1.04f, 0.64f}, {64, 32, 4, 1, 3.0f, 1.08f, 0.70f},
    {64, 64, 4, 3, 4.0f, 1.40f, 3.34f}, {64, 64, 1, 3, 4.0f, 0.46f, 0.64f}, {128, 128, 1, 1, 4.5f, 0.86f, 0.50f},
    {256, 256, 1, 1, 8.5f, 1.58f, 2.00f},
};

inline float mx_cost(int form, uint64_t M, uint64_t N, uint64_t K, uint64_t cus) {
    const MxCost &c = MX_COST[form];
    const uint64_t wgs = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const uint64_t steps = ((K + 255) / 256 + c.step - 1) / c.step;
    if (wgs <= cus) return c.start + c.one * (float)steps;
    return (float)((wgs + cus * c.per_cu - 1) / (cus * c.per_cu)) * (c.start + c.more * (float)steps);
}

// For more than one row.
inline MxForm mx_pick(uint64_t M, uint64_t N, uint64_t K, uint64_t cus) {
    int best = 0;
    float us = -1.0f;
    for (int f = 0; f < MX_FORMS; ++f) {
        if (MX_COST[f].bm >= 4 * M && MX_COST[f].bm > 16) continue;   // a tile holds more than a quarter of its rows
        const float t = mx_cost(f, M, N, K, cus);
        if (us < 0.0f || t < us) us = t, best = f;
    }
    return (MxForm)best;
}

}  // namespace reng
