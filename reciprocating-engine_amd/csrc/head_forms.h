// head_forms.h - how many heads a group of lanes of the head norms
// (csrc/head_norm_rope.hip) takes. Plain C++ so that the host tests can check the
// rule with the code the launcher runs.
#pragma once

#include <stdint.h>

namespace reng {

// Workgroups of a token, of `group` heads or of four times that.
inline uint32_t head_parts(uint32_t heads, uint32_t group, bool four) {
    return (heads + (four ? 4 : 1) * group - 1) / ((four ? 4 : 1) * group);
}
constexpr uint64_t HEAD_LAUNCH = 1u << 24;   // workgroups of a launch, of 256 threads

// Four heads a group of lanes read the token's sines and cosines once, in a quarter of the workgroups. That pays
// once there are two and a half of those a CU, and as far as they waste few groups of lanes (a third more than one
// head each takes). Times of four for one, us, rotated by one axis or by several a run of eight pairs: 56 heads of
// 128 (16 groups for 16) 384 tokens 6.7 for 6.3, 512 7.4 for 7.5, 640 8.8 for 9.7, 1024 10.7 for 12.1, 4096 25.5
// for 31.0; 36 heads (16 for 12) 512 tokens 6.3 for 6.0, 768 7.4 for 8.4, 4096 21.2 for 23.1 (by one axis such
// shares are equal, within 7% either way); 80 (32 for 20) 5 to 15% slower at every number. Axes in turn pair by
// pair load eight positions: from one and a half workgroups a CU on, with three fifths more groups (36 heads 384
// tokens 6.9 for 7.3, 80 heads 1024 tokens 18.4 for 21.8). Without tables there is nothing to share: 56 heads
// within 5% either way, 80 20% slower.
inline bool heads_by_four(uint64_t tokens, uint32_t heads, uint32_t group, bool rotates, bool mixed, uint64_t cus) {
    const uint32_t one = head_parts(heads, group, false), four = head_parts(heads, group, true);
    if (tokens * one >= HEAD_LAUNCH) return true;
    return 2 * one >= (mixed ? 5 : rotates ? 6 : 8) * four && 2 * tokens * four >= (mixed ? 3 : 5) * cus;
}

}  // namespace reng
