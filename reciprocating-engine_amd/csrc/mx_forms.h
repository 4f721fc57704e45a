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

// Outputs of a workgroup, stages of 256 k that it takes a step, and times (us): the start and a step of a
// CU's first workgroup, and what each further one of that CU adds to them. Fitted to graph-replayed
// timings of every form on 156 products (M 2 to 6000, N 1024 to 27648, K 576 to 27648); on these the
// choice is the fastest form or within 6% of it (0.3% in the mean). The weight's bytes are no term of
// their own, so for wider ones its times are too short, and the order less sure: on 75 products of N 49152
// to 152064 (M 2 to 1024) the choice is 3.6% from the fastest in the mean, 19% at most but for 17 and 24 rows
// [65536, 8192], 28% and 25%.
struct MxCost {
    uint32_t bm, bn, step;
    float start, start_more, one, more;
};
constexpr MxCost MX_COST[MX_FORMS] = {
    {16, 16, 4, 2.94f, 0.38f, 0.41f, 0.31f}, {16, 32, 4, 3.00f, 1.32f, 0.52f, 0.55f}, {32, 16, 4, 3.01f, 0.96f, 0.51f, 0.45f},
    {32, 32, 4, 2.81f, 0.61f, 0.70f, 0.54f}, {64, 16, 4, 3.23f, 1.11f, 0.73f, 0.67f}, {64, 32, 4, 3.25f, 1.73f, 0.94f, 0.78f},
    {64, 64, 4, 3.71f, 2.75f, 1.46f, 1.09f}, {64, 64, 1, 3.57f, 1.08f, 0.45f, 0.20f}, {128, 128, 1, 3.66f, 0.78f, 0.82f, 0.58f},
    {256, 256, 1, 12.11f, 13.75f, 1.46f, 1.42f},
};

inline float mx_cost(int form, uint64_t M, uint64_t N, uint64_t K, uint64_t cus) {
    const MxCost &c = MX_COST[form];
    const uint64_t wgs = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const float further = (float)((wgs + cus - 1) / cus - 1), steps = (float)(((K + 255) / 256 + c.step - 1) / c.step);
    return c.start + c.start_more * further + steps * (c.one + c.more * further);
}

// One row: rows of b that a wave takes, and k of a piece. The waves that share rows and take pieces in
// turn: enough for sixteen waves a CU, where there are as many pieces (eight: [4096, 14336] 9.8 us for 8.9).
constexpr uint32_t MX_ROW_NR = 2, MX_ROW_K = 2048;
inline uint32_t mx_row_waves(uint64_t N, uint64_t K, uint64_t cus) {
    const uint64_t groups = (N + MX_ROW_NR - 1) / MX_ROW_NR, pieces = (K + MX_ROW_K - 1) / MX_ROW_K, want = cus * 16;
    return groups >= want || pieces < 2 ? 1 : groups * 2 >= want || pieces < 4 ? 2 : 4;
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
