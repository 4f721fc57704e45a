// head_norm_rope.hip - norms of queries and keys per head, the rotation of their
// positions and the write of keys and values, as bf16 rows or into a 4-bit cache, in
// one pass:
//
//   y = x / sqrt(mean(x^2) + eps) * gamma        (per head; queries and keys)
//   y[d], y[d + half] = rotate(y[d], y[d + half]) by row positions[axis(d), token] of the tables
//
// in f32, rounded once, to bf16 or to e2m1 under the scale of 32 values (mx.h).
//
// A group of lanes takes one head of one token, eight values each: the norm's sum and the
// block maxima are lane exchanges, a rotation's other value is one too. Consecutive
// groups take consecutive heads, so a token's row is read as it lies. Of a rotation's tables a
// lane reads its dimensions' entries once a token, whatever the heads it goes through.
//
// What bounds it: the launch and a chain of loads, position then table, for few tokens (one 3.8 us); for
// many too while they are one round of workgroups (1024 of 56 heads of 128, 31 MB: 12.7 us, 2.5 TB/s),
// HBM beyond (4096: 31.8 us, 3.8 TB/s; a copy reaches 5.1).
#include "head_forms.h"
#include "mx.h"

namespace reng {
namespace {

using namespace mx;

struct HeadsArgs {
    const uint16_t *q, *k, *v;
    size_t q_ld, kv_ld;
    uint32_t tokens, nh, nkv, hd;
    const float *q_gamma, *k_gamma;
    float eps;
    const float *sin_table, *cos_table;   // null: no rotation
    uint32_t table_rows, rot;
    const int32_t *positions;
    uint16_t *q_out, *k_rows, *v_rows;
    reng_hip_mx_cache cache;
    size_t first;
    uint64_t axes8;       // of each 8 pairs their axis, four bits; MIXED: pair_axis says it pair by pair
    bool mixed;           // whether some are
    uint8_t pair_axis[128];
};
constexpr uint32_t MIXED = 15;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <bool VEC>
__device__ __forceinline__ u32x4_t load8(const uint16_t *p) {
    if constexpr (VEC) return *reinterpret_cast<const u32x4_t *>(p);
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return v;
}

template <bool VEC>
__device__ __forceinline__ void store8(uint16_t *p, const float (&x)[8]) {
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, bf16x2));
    if constexpr (VEC) {
        *reinterpret_cast<u32x4_t *>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
    }
}

__device__ __forceinline__ void load8f(const float *p, float (&x)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float4 v = reinterpret_cast<const float4 *>(p)[h];
        x[4 * h] = v.x, x[4 * h + 1] = v.y, x[4 * h + 2] = v.z, x[4 * h + 3] = v.w;
    }
}

// The sines and cosines of values d .. d + 7, whose pairs start at `pair`.
__device__ __forceinline__ void tables(const HeadsArgs &a, uint32_t token, uint32_t d, uint32_t pair, float (&sn)[8],
                                       float (&cs)[8]) {
    auto row_of = [&](uint32_t axis) { return (uint32_t)a.positions[(size_t)axis * a.tokens + token]; };
    // A row outside the tables is read as row 0 and then made NaN, without a branch on the position.
    const uint32_t axis = (uint32_t)(a.axes8 >> (pair / 2)) & 15;
    if (axis != MIXED) {
        const uint32_t row = row_of(axis);
        const bool in = row < a.table_rows;
        const size_t at = (size_t)(in ? row : 0) * a.rot + d;
        load8f(a.sin_table + at, sn);
        load8f(a.cos_table + at, cs);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sn[i] = in ? sn[i] : __builtin_nanf("");
            cs[i] = in ? cs[i] : __builtin_nanf("");
        }
    } else {
        uint32_t row[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) row[i] = row_of(a.pair_axis[pair + i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool in = row[i] < a.table_rows;
            const size_t at = (size_t)(in ? row[i] : 0) * a.rot + d + i;
            const float x = a.sin_table[at], y = a.cos_table[at];
            sn[i] = in ? x : __builtin_nanf("");
            cs[i] = in ? y : __builtin_nanf("");
        }
    }
}

// The value of lane ^ (L / 2) of a group of L; for 16 lanes without LDS.
template <int L>
__device__ __forceinline__ float across(float v) {
    if constexpr (L == 16)   // row_ror:8
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, true));
    return __shfl_xor(v, L / 2, 64);
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    v += across<L>(v);
    if constexpr (L == 16) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, true));   // row_ror:4
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, true));   // row_ror:2
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, true));   // row_ror:1
    } else {
#pragma unroll
        for (int o = L / 4; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    }
    return v;
}

// L lanes a head: 4, 8, 16 or 32, at least hd / 8. A workgroup takes IT times 256 / L heads of a token, whose
// rows and the token's sines and cosines are asked for at once. VEC: 16-byte aligned rows. MX: into the cache.
template <int L, int IT, bool VEC, bool MX>
__global__ __launch_bounds__(256) void head_norm_rope(const HeadsArgs a, uint32_t parts) {
    constexpr uint32_t G = 256 / L;
    const uint32_t lane = threadIdx.x & 63, li = threadIdx.x % L, heads = a.nh + 2 * a.nkv;
    const uint32_t token = blockIdx.x / parts, h0 = blockIdx.x % parts * (IT * G) + threadIdx.x / L;
    const bool has = li * 8 < a.hd;   // a lane without values still takes part in the exchanges, with zeros
    const uint32_t d = has ? li * 8 : 0;
    struct Head {
        uint32_t part, g;   // q, k or v, and which of its heads
    };
    auto head_of = [&](uint32_t h) {
        return h < a.nh ? Head{0, h} : h < a.nh + a.nkv ? Head{1, h - a.nh} : Head{2, h - a.nh - a.nkv};
    };
    u32x4_t raw[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {   // past the last head the last one again, which is not stored
        const Head h = head_of(min(h0 + it * G, heads - 1));
        const uint16_t *base = h.part == 0 ? a.q : h.part == 2 && a.v ? a.v : a.k;
        raw[it] = load8<VEC>(base + (size_t)token * (h.part == 0 ? a.q_ld : a.kv_ld) + h.g * a.hd + d);
        if (a.hd != 8 * L && !has) raw[it] = u32x4_t{0u, 0u, 0u, 0u};
    }
    const uint32_t half = a.rot / 2;
    const bool low = d < half, turns = a.sin_table && d < a.rot, whole = a.rot == 8 * L;
    float gq[8], gk[8], sn[8], cs[8];
    if (turns) tables(a, token, d, low ? d : d - half, sn, cs);
    if (a.q_gamma)
#pragma unroll
        for (int i = 0; i < 8; ++i) gq[i] = a.q_gamma[d + i];
    if (a.k_gamma)
#pragma unroll
        for (int i = 0; i < 8; ++i) gk[i] = a.k_gamma[d + i];
    // y[d] = x[d] cos - x[d + half] sin, y[d + half] = x[d + half] cos + x[d] sin
#pragma unroll
    for (int i = 0; i < 8; ++i) sn[i] = low ? -sn[i] : sn[i];
    const uint32_t other = low ? lane + half / 8 : lane - half / 8;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const bool on = has && h0 + it * G < heads;
        const Head h = head_of(min(h0 + it * G, heads - 1));
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(raw[it][i] << 16);
            x[2 * i + 1] = __uint_as_float(raw[it][i] & 0xffff0000u);
        }
        if (a.q_gamma || a.k_gamma) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
            ss = group_sum<L>(ss);
            const float inv = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
            if (h.part == 0 && a.q_gamma)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * gq[i];
            if (h.part == 1 && a.k_gamma)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * gk[i];
        }
        if (a.sin_table) {
            float y[8];
            if (whole)
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = across<L>(x[i]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], (int)other, 64);
            if (turns && h.part < 2)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], cs[i], y[i] * sn[i]);
        }
        if (!MX || h.part == 0) {
            uint16_t *out = h.part == 0 ? a.q_out : h.part == 1 ? a.k_rows : a.v_rows;
            if (on && out) store8<VEC>(out + (size_t)token * ((h.part == 0 ? a.nh : a.nkv) * a.hd) + h.g * a.hd + d, x);
        }
        if constexpr (MX) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
            const uint32_t top = quad_max(m), byte = has ? scale_byte(top) : ONE_BYTE;
            uint32_t word;
            if constexpr (L >= 16) {
                word = scale_word(byte);
            } else {   // one or two blocks
                word = byte << (8 * (li / 4));
                if constexpr (L == 8) word |= (uint32_t)__builtin_amdgcn_ds_swizzle((int)word, 0x101f);   // lane ^ 4
                word |= L == 8 ? 0x7f7f0000u : 0x7f7f7f00u;
            }
            if (on && h.part > 0) {
                const size_t row = (size_t)h.g * a.cache.capacity + a.first + token, sp = scale_pitch(a.hd);
                uint8_t *codes = h.part == 1 ? a.cache.k_codes : a.cache.v_codes;
                uint8_t *scales = h.part == 1 ? a.cache.k_scales : a.cache.v_scales;
                *reinterpret_cast<uint32_t *>(codes + row * (a.hd / 2) + d / 2) = encode8(x, byte);
                if (li % 16 == 0) *reinterpret_cast<uint32_t *>(scales + row * sp + li / 4) = word;
            }
        }
    }
}

template <int L, bool VEC, bool MX>
int launch_lanes(const HeadsArgs &a, hipStream_t st) {
    const uint32_t heads = a.nh + 2 * a.nkv;
    constexpr uint32_t G = 256 / L;
    const bool four = heads_by_four(a.tokens, heads, G, a.sin_table, a.mixed, (uint64_t)device_props().cus);
    const uint32_t parts = head_parts(heads, G, four);
    RENG_REQUIRE((uint64_t)a.tokens * parts < HEAD_LAUNCH, "%u tokens of %u heads are too many for a launch", a.tokens, heads);
    const auto kern = four ? head_norm_rope<L, 4, VEC, MX> : head_norm_rope<L, 1, VEC, MX>;
    hipLaunchKernelGGL(kern, dim3(a.tokens * parts), dim3(256), 0, st, a, parts);
    return check_launch("head_norm_rope");
}

template <bool MX>
int launch_heads(const HeadsArgs &a, bool vec, hipStream_t st) {
    if (a.hd <= 32) return vec ? launch_lanes<4, true, MX>(a, st) : launch_lanes<4, false, MX>(a, st);
    if (a.hd <= 64) return vec ? launch_lanes<8, true, MX>(a, st) : launch_lanes<8, false, MX>(a, st);
    if (a.hd <= 128) return vec ? launch_lanes<16, true, MX>(a, st) : launch_lanes<16, false, MX>(a, st);
    return vec ? launch_lanes<32, true, MX>(a, st) : launch_lanes<32, false, MX>(a, st);
}

// What both entry points check and fill in.
int heads_args(HeadsArgs &a, const uint16_t *q, size_t q_ld, const uint16_t *k, const uint16_t *v, size_t kv_ld,
               size_t tokens, size_t nh, size_t nkv, size_t hd, const float *q_gamma, const float *k_gamma, float eps,
               const reng_hip_rope *rope, const int32_t *positions, uint16_t *q_out) {
    RENG_REQUIRE(tokens >= 1 && tokens < (1u << 22), "%zu tokens; expected 1 to 2^22 - 1", tokens);
    RENG_REQUIRE(nh <= 4096 && nkv >= 1 && nkv <= 4096,
                 "%zu query and %zu key/value heads; at most 4096 of each, one key/value head or more", nh, nkv);
    RENG_REQUIRE(hd >= 32 && hd % 32 == 0 && hd <= 256, "head_dim %zu is no multiple of 32 in [32, 256]", hd);
    RENG_REQUIRE(nh == 0 ? !q && !q_out : q && q_out, "%zu query heads, and their pointers are%s null", nh, nh ? "" : " not");
    RENG_REQUIRE(k, "null pointer");
    RENG_REQUIRE(nh == 0 || q_ld >= nh * hd, "query row pitch %zu is below %zu values", q_ld, nh * hd);
    RENG_REQUIRE(kv_ld >= nkv * hd, "key/value row pitch %zu is below %zu values", kv_ld, nkv * hd);
    RENG_REQUIRE(q_ld < (1u << 31) && kv_ld < (1u << 31), "dimension too large");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                   reinterpret_cast<uintptr_t>(q_out)) & 1) == 0 &&
                     ((reinterpret_cast<uintptr_t>(q_gamma) | reinterpret_cast<uintptr_t>(k_gamma) |
                       reinterpret_cast<uintptr_t>(positions)) & 3) == 0,
                 "a pointer is not aligned to its elements");
    RENG_REQUIRE(eps >= 0.0f && eps < __builtin_inff(), "eps is not finite and at least 0");
    a.q = q, a.k = k, a.v = v, a.q_ld = q_ld, a.kv_ld = kv_ld;
    a.tokens = (uint32_t)tokens, a.nh = (uint32_t)nh, a.nkv = (uint32_t)nkv, a.hd = (uint32_t)hd;
    a.q_gamma = q_gamma, a.k_gamma = k_gamma, a.eps = eps, a.q_out = q_out;
    a.sin_table = a.cos_table = nullptr;
    a.axes8 = 0;
    if (!rope) return RENG_HIP_OK;
    const reng_hip_rope &r = *rope;
    RENG_REQUIRE(r.rot_dim >= 16 && r.rot_dim % 16 == 0 && r.rot_dim <= hd, "rot_dim %zu is no multiple of 16 in [16, %zu]",
                 r.rot_dim, hd);
    RENG_REQUIRE(r.axes >= 1 && r.axes <= RENG_HIP_ROPE_MAX_AXES, "%zu axes; expected 1 to %d", r.axes, RENG_HIP_ROPE_MAX_AXES);
    RENG_REQUIRE(r.table_rows >= 1 && r.table_rows < (1u << 31), "tables of %zu rows; expected 1 to 2^31 - 1", r.table_rows);
    RENG_REQUIRE(r.sin_table && r.cos_table && positions, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(r.sin_table) | reinterpret_cast<uintptr_t>(r.cos_table)) & 15) == 0,
                 "tables must be 16-byte aligned");
    if (r.pair_axis)
        for (size_t i = 0; i < r.rot_dim / 2; ++i)
            RENG_REQUIRE(r.pair_axis[i] < r.axes, "pair %zu has axis %d of %zu", i, r.pair_axis[i], r.axes);
    a.sin_table = r.sin_table, a.cos_table = r.cos_table, a.table_rows = (uint32_t)r.table_rows;
    a.rot = (uint32_t)r.rot_dim, a.positions = positions;
    if (r.pair_axis)
        for (size_t i = 0; i < r.rot_dim / 2; ++i) {
            a.pair_axis[i] = r.pair_axis[i];
            const uint64_t eight = r.pair_axis[i / 8 * 8] == r.pair_axis[i] ? r.pair_axis[i] : MIXED;
            a.axes8 |= eight << (i / 8 * 4);
            a.mixed |= eight == MIXED;
        }
    return RENG_HIP_OK;
}

bool rows_aligned(const HeadsArgs &a) {
    return ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
             reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k_rows) |
             reinterpret_cast<uintptr_t>(a.v_rows)) & 15) == 0 &&
           (a.nh == 0 || a.q_ld % 8 == 0) && a.kv_ld % 8 == 0;
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API int reng_hip_head_norm_rope_bf16(const uint16_t *q, size_t q_ld, const uint16_t *k, const uint16_t *v,
                                              size_t kv_ld, size_t tokens, size_t n_heads, size_t n_kv_heads,
                                              size_t head_dim, const float *q_gamma, const float *k_gamma, float eps,
                                              const reng_hip_rope *rope, const int32_t *positions, uint16_t *q_out,
                                              uint16_t *k_rows, uint16_t *v_rows, void *stream) {
    clear_error();
    HeadsArgs a{};
    if (int rc = heads_args(a, q, q_ld, k, v, kv_ld, tokens, n_heads, n_kv_heads, head_dim, q_gamma, k_gamma, eps, rope,
                            positions, q_out))
        return rc;
    RENG_REQUIRE(k_rows && !v == !v_rows, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(k_rows) | reinterpret_cast<uintptr_t>(v_rows)) & 1) == 0,
                 "a pointer is not aligned to its elements");
    a.k_rows = k_rows, a.v_rows = v_rows;
    return launch_heads<false>(a, rows_aligned(a), static_cast<hipStream_t>(stream));
}

RENG_HIP_API int reng_hip_head_norm_rope_mxfp4(const uint16_t *q, size_t q_ld, const uint16_t *k, const uint16_t *v,
                                               size_t kv_ld, size_t tokens, size_t n_heads, const float *q_gamma,
                                               const float *k_gamma, float eps, const reng_hip_rope *rope,
                                               const int32_t *positions, uint16_t *q_out, const reng_hip_mx_cache *cache,
                                               size_t first, void *stream) {
    clear_error();
    if (int rc = check_mx_cache(cache)) return rc;
    HeadsArgs a{};
    if (int rc = heads_args(a, q, q_ld, k, v, kv_ld, tokens, n_heads, cache->n_kv_heads, cache->head_dim, q_gamma, k_gamma,
                            eps, rope, positions, q_out))
        return rc;
    RENG_REQUIRE(v, "null pointer");
    RENG_REQUIRE(first <= cache->capacity && tokens <= cache->capacity - first, "rows %zu .. %zu of a cache of %zu", first,
                 first + tokens, cache->capacity);
    a.cache = *cache, a.first = first;
    return launch_heads<true>(a, rows_aligned(a), static_cast<hipStream_t>(stream));
}
