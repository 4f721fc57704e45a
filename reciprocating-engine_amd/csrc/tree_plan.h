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

// rows: query rows of a key/value head, tokens x heads that share it.
inline TreePlan tree_plan(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, bool aligned, size_t cus) {
    TreePlan p{};
    p.fast = hd % 8 == 0 && hd <= 256 && aligned;
    p.splits = 1;
    if (!p.fast) return p;
    p.hdp = hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256;
    const size_t rows = tokens * (nh / nkv), cache = len + tokens;
    const int forms = p.hdp == 256 ? 3 : 4;
    while (p.form + 1 < forms && rows > 32 * tree_form(p.hdp, p.form).rw) ++p.form;
    // FORM CHOSEN
    const TreeForm f = tree_form(p.hdp, p.form);
    p.row_blocks = (uint32_t)((rows + 32 * f.rw - 1) / (32 * f.rw));
    p.tiles = (uint32_t)((cache + f.tk - 1) / f.tk);
    // Workgroups for every CU, but two steps of tiles a workgroup at least.
    const size_t wgs = nkv * p.row_blocks;
    size_t s = (cus + wgs - 1) / wgs;
    const size_t most = p.tiles / (2 * f.kw);
    if (s > most) s = most;
    if (s > TREE_SPLIT_MAX) s = TREE_SPLIT_MAX;
    p.splits = s < 1 ? 1 : (uint32_t)s;
    // SPLITS CHOSEN
    return p;
}

// What a wave leaves of a split: for 32 rows the unnormalised outputs, as its 64 lanes hold
// them, and each lane's maximum and sum.
#if defined(__HIPCC__)
__host__ __device__
#endif
constexpr uint32_t tree_wave_floats(uint32_t hdp) { return hdp * 32 + 128; }

inline size_t tree_part_bytes(const TreePlan &p, size_t nkv) {
    return p.splits < 2 ? 0
                        : (size_t)p.splits * nkv * p.row_blocks * tree_form(p.hdp, p.form).rw *
                              tree_wave_floats(p.hdp) * sizeof(float);
}

// The most tree_part_bytes asks for over 1 .. tokens tokens and 0 .. len context
// rows: with the form and the row blocks given the splits only grow with the rows,
// so the most tokens of each (form, row blocks) are looked at.
inline size_t tree_workspace(size_t nh, size_t nkv, size_t hd, size_t len, size_t tokens, size_t cus) {
    size_t most = 0;
    const size_t per = nh / nkv;
    auto at = [&](size_t t) {
        if (t > tokens) t = tokens;
        const TreePlan p = tree_plan(nh, nkv, hd, len, t, true, cus);
        const size_t b = tree_part_bytes(p, nkv);
        if (b > most) most = b;
        return p;
    };
    const TreePlan last = at(tokens);
    if (!last.fast) return 0;
    for (int f = 0; f < last.form; ++f)
        if (const size_t t = 32 * tree_form(last.hdp, f).rw / per) at(t);
    const size_t block = 32 * tree_form(last.hdp, last.form).rw;
    for (uint32_t rb = 1; rb < last.row_blocks && nkv * rb < cus; ++rb)
        if (const size_t t = rb * block / per) at(t);
    return most;
}

}  // namespace reng
