// attention_mxfp4.hip - attention of a chain or tree of tokens over a cache held in
// 4 bits (mx.h), read as it lies:
//
//   s_j = scale * q[i, h] . k[j, g]        p = softmax(s)        out[i, h] = sum_j p_j v[j, g]
//
// per token i and query head h, g = h / (n_heads / n_kv_heads), over the rows j that the
// token sees: the context's len, and of the tokens' own those of its mask row, or without
// a mask rows 0 .. i. A code times its scale is a bf16 value exactly, so nothing is
// rounded on the way to the matrix cores.
//
// The query rows of a key/value head (row r: token r / per, query head r % per of the per
// that share it) go 16 to a tile and QT tiles to a wave; the four waves of a workgroup take
// tiles of 32 cache rows in turn, and merge in LDS; splits of the cache merge in a second
// kernel (mx_attention_plan.h). A wave needs nothing of the others until then.
//
// Per tile a wave forms S^T = K Q^T on v_mfma_f32_16x16x32_bf16. Lane l has key l % 16 and,
// of its dimensions, the quarter l / 16: the order in which dimensions are summed is free, so
// a lane's codes are consecutive bytes and lie under one scale (two of 256 dimensions), and the
// queries' registers follow that order. The results have query l % 16 and four keys from
// 4 (l / 16), which is how O^T = V^T P^T takes the weights. V^T comes from LDS, where a
// wave puts a tile's values as bf16, by transposing reads.
//
// A row whose key or value holds a scale from 253 on (NaN, or magnitudes bf16 ends at) counts as NaN: its
// key's scale becomes NaN and its value's 1, so that its score decides who meets it, and a
// weight of 0 takes nothing from a value.
#include "common.h"
#include "mx.h"
#include "mx_attention_plan.h"

namespace reng {
namespace {

using namespace mx;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct MxAttn {
    const uint16_t *q;
    const uint8_t *kc, *ks, *vc, *vs;
    size_t cap;             // rows of a head
    uint32_t nh, nkv, hd, sp;
    uint32_t len, tokens;
    const uint32_t *mask;   // null: a chain
    uint32_t words;         // of a mask row
    float scale;
    uint16_t *out;
    uint32_t row_blocks, units, splits, base, more;   // split s: base tiles, one more for the first `more`
    float *part;            // null: one pass
};

// Bit b: whether token i sees cache row j0 + b.
__device__ __forceinline__ uint32_t seen_bits(const MxAttn &a, uint32_t i, uint32_t j0) {
    const int d0 = (int)j0 - (int)a.len;
    const int n = (a.mask ? (int)a.tokens : (int)i + 1) - d0;   // rows j0 .. j0 + n - 1 may be seen
    uint32_t w = 0xffffffffu;
    if (a.mask) {
        const uint32_t *m = a.mask + (size_t)i * a.words;
        if (d0 >= 0) {
            const uint32_t k = (uint32_t)d0 / 32, sh = (uint32_t)d0 % 32;
            const uint32_t lo = k < a.words ? m[k] : 0u, hi = k + 1 < a.words ? m[k + 1] : 0u;
            w = (uint32_t)((((uint64_t)hi << 32) | lo) >> sh);
        } else if (d0 > -32) {
            w = (m[0] << -d0) | ((1u << -d0) - 1u);
        }
    }
    if (n < 32) w &= n <= 0 ? 0u : (1u << n) - 1u;
    return w;
}

__device__ bool sees_any(const MxAttn &a, uint32_t i) {
    if (a.len || !a.mask) return true;
    uint32_t any = 0;
    for (uint32_t w = 0; w < a.words; ++w) {
        const uint32_t left = a.tokens - 32 * w;   // bits from tokens on are not read
        any |= a.mask[(size_t)i * a.words + w] & (left < 32 ? (1u << left) - 1u : 0xffffffffu);
    }
    return any != 0;
}

__device__ __forceinline__ u32x2 read_tr(const uint8_t *p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4 *)p));
}

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
}

// Over the four lanes of a query (16 apart).
__device__ __forceinline__ float query_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float query_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// o / l as bf16; l = 0: nothing seen gives zeros, scores that are all -inf give NaN.
__device__ __forceinline__ u32x2 finish(const f32x4 &o, float l, bool any) {
    if (!any) return u32x2{0u, 0u};
    const float r = 1.0f / l;   // one rounding more than a division, far below bf16's
    return u32x2{pack_bf16(o.x * r, o.y * r), pack_bf16(o.z * r, o.w * r)};
}

// The slot of 16-byte chunk c of a tile's row r. Eight consecutive rows written at one chunk
// and four read over two chunks lie in different slots.
__device__ __forceinline__ uint32_t value_slot(uint32_t r, uint32_t c) {
    return c ^ (((r & 3) << 1) | ((r >> 2) & 1));
}

template <int HD, int QT>
__global__ __launch_bounds__(64 * MXA_WAVES) void attention_mxfp4(const MxAttn a) {
    constexpr int NW = MXA_WAVES, ST = HD / 32, DT = HD / 16;   // products a score; tiles of dimensions
    constexpr int LB = HD / 8, CH = LB <= 16 ? 1 : LB / 16;     // bytes of a lane; 16-byte chunks of them
    constexpr int ROWB = 2 * HD, VBUF = MXA_TILE * ROWB;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float ml[2][NW][16];
    // Workgroups go to the XCDs in turn: the row blocks of one split and key/value head
    // follow each other on one XCD, whose L2 gives them the rows after the first.
    const uint32_t b = blockIdx.x / MXA_XCDS, rb = b % a.row_blocks;
    const uint32_t unit = b / a.row_blocks * MXA_XCDS + blockIdx.x % MXA_XCDS;
    if (unit >= a.units) return;
    const uint32_t g = unit % a.nkv, split = unit / a.nkv;
    const uint32_t lane = threadIdx.x & 63, r16 = lane & 15, q4 = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, rows = a.len + a.tokens;
    uint8_t *vbuf = lds + wave * VBUF;

    // This lane's query rows (clamped: rows past the last are not stored).
    // scale < 0 goes into the queries' signs, so that the largest product is the largest score.
    const float c = fabsf(a.scale) * 1.44269504088896341f;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    uint32_t tok[QT];
    u32x4 qf[QT][ST];
    const uint32_t dim0 = q4 * (HD / 4);   // this lane's dimensions
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const uint32_t r = min((rb * QT + t) * 16 + r16, R - 1);
        tok[t] = r / per;
        const uint16_t *qr = a.q + ((size_t)tok[t] * a.nh + g * per + r % per) * a.hd;
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            u32x4 v{0u, 0u, 0u, 0u};
            if (dim0 + 8 * s < a.hd) v = *reinterpret_cast<const u32x4 *>(qr + dim0 + 8 * s);
            qf[t][s] = v ^ flip;
        }
    }

    // The split's tiles, cut for a chain at the last row its tokens see.
    const uint32_t t0 = split * a.base + min(split, a.more);
    uint32_t t1 = t0 + a.base + (split < a.more);
    if (!a.mask) {
        const uint32_t last = min((rb * QT + QT) * 16 - 1, R - 1) / per;
        t1 = min(t1, (a.len + last) / MXA_TILE + 1);
    }

    const size_t head = (size_t)g * a.cap;
    const uint32_t rowb = a.hd / 2;
    struct Codes {
        uint32_t w[LB / 4];
        uint32_t s[CH];   // scale bytes
    };
    // Row j's codes of this lane; zeros past the head's dimensions.
    auto load = [&](const uint8_t *codes, const uint8_t *scales, uint32_t j) __attribute__((always_inline)) {
        const size_t row = head + min(j, rows - 1);
        Codes v;
        const uint8_t *p = codes + row * rowb + dim0 / 2, *s = scales + row * a.sp + dim0 / 32;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const bool on = dim0 + 32 * i < a.hd;
            v.s[i] = on ? s[i] : ONE_BYTE;
            if constexpr (LB == 8) {
                const u32x2 x = on ? *reinterpret_cast<const u32x2 *>(p) : u32x2{0u, 0u};
                v.w[0] = x.x, v.w[1] = x.y;
            } else {
                const u32x4 x = on ? reinterpret_cast<const u32x4 *>(p)[i] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 4; ++e) v.w[4 * i + e] = x[e];
            }
        }
        return v;
    };

    f32x4 o[DT][QT];
    float m[QT], l[QT];   // the running maximum of the products, this lane's share of the sum
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = -INFINITY, l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d][t] = f32x4{0, 0, 0, 0};
    }
    for (uint32_t tile = t0 + wave; tile < t1; tile += NW) {
        const uint32_t j0 = tile * MXA_TILE;
        f32x4 s[2][QT];
#pragma unroll
        for (int u = 0; u < 2; ++u) {   // keys 16 u ..
            Codes k = load(a.kc, a.ks, j0 + 16 * u + r16), v = load(a.vc, a.vs, j0 + 16 * u + r16);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const bool odd = max(k.s[i], v.s[i]) >= 253;
                k.s[i] = odd ? NAN_BYTE : k.s[i];
                v.s[i] = odd ? ONE_BYTE : v.s[i];
            }
            const uint32_t row = 16 * u + r16;
#pragma unroll
            for (int e = 0; e < ST; ++e)
                *reinterpret_cast<u32x4 *>(vbuf + row * ROWB + 16 * value_slot(row, dim0 / 8 + e)) =
                    decode8(v.w[e], scale_operand(v.s[e * CH / ST]));
#pragma unroll
            for (int t = 0; t < QT; ++t) s[u][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < ST; ++e) {
                const bf16x8 kf = __builtin_bit_cast(bf16x8, decode8(k.w[e], scale_operand(k.s[e * CH / ST])));
#pragma unroll
                for (int t = 0; t < QT; ++t)
                    s[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, __builtin_bit_cast(bf16x8, qf[t][e]), s[u][t], 0, 0, 0);
            }
        }
        asm volatile("" ::: "memory");   // the values are read by other lanes than wrote them, in the wave's own order
        const bool masked = j0 + MXA_TILE > a.len;
        u32x4 pw[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            uint32_t see = 0xffffffffu;
            if (masked) {
                see = seen_bits(a, tok[t], j0) >> (4 * q4);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!((see >> (16 * (i / 4) + i % 4)) & 1)) s[i / 4][t][i % 4] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0][t][0], s[0][t][1]), fmaxf(s[0][t][2], s[0][t][3])),
                             fmaxf(fmaxf(s[1][t][0], s[1][t][1]), fmaxf(s[1][t][2], s[1][t][3])));
            // The maximum moves, and what is summed so far is scaled down, only where a
            // score passes it by more than 2^8: weights up to 256 lose nothing in f32 or bf16.
            if (__builtin_amdgcn_ballot_w64((mx - m[t]) * c > 8.0f || (m[t] == -INFINITY && mx > m[t]))) {
                mx = query_max(mx);
                const bool move = (mx - m[t]) * c > 8.0f || (m[t] == -INFINITY && mx > m[t]);
                const float f = !move ? 1.0f : m[t] == -INFINITY ? 0.0f : exp2f((m[t] - mx) * c);
                if (move) m[t] = mx;
                l[t] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][t] *= f;
            }
            // With nothing above -inf so far, exponents are taken against 0: they are 0.
            const float mc = m[t] == -INFINITY ? 0.0f : m[t] * c;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][t][i % 4], c, -mc));
                if (masked) p[i] = (see >> (16 * (i / 4) + i % 4)) & 1 ? p[i] : 0.0f;
                l[t] += p[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) pw[t][i] = pack_bf16(p[2 * i], p[2 * i + 1]);
        }
        // V^T of the tile's rows in the order of the weights. Lane: dimensions 4 (l % 4) .. + 3 of a row.
        const uint32_t row = 4 * q4 + r16 / 4;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const uint32_t ch = 2 * d + (r16 & 3) / 2, in = 8 * (r16 & 1);
            const u32x2 v0 = read_tr(vbuf + row * ROWB + 16 * value_slot(row, ch) + in);
            const u32x2 v1 = read_tr(vbuf + (row + 16) * ROWB + 16 * value_slot(row + 16, ch) + in);
            const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{v0.x, v0.y, v1.x, v1.y});
#pragma unroll
            for (int t = 0; t < QT; ++t)
                o[d][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, pw[t]), o[d][t], 0, 0, 0);
        }
        asm volatile("" ::: "memory");
    }

    // The waves' (o, m, l) through LDS, a query tile at a time: a wave merges a quarter of its dimensions.
    constexpr int MD = DT / NW;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        __syncthreads();
        const float sum = query_sum(l[t]), top_c = m[t] == -INFINITY ? -INFINITY : m[t] * c;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(vbuf + d * 1024 + lane * 16) = o[d][t];
        if (q4 == 0) ml[0][wave][r16] = top_c, ml[1][wave][r16] = sum;
        __syncthreads();
        float top = ml[0][0][r16];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, ml[0][w][r16]);
        const float at = top == -INFINITY ? 0.0f : top;
        float all = 0.0f;
        f32x4 x[MD];
#pragma unroll
        for (int d = 0; d < MD; ++d) x[d] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = exp2f(ml[0][w][r16] - at);
            all += ml[1][w][r16] * f;
#pragma unroll
            for (int d = 0; d < MD; ++d)
                x[d] += *reinterpret_cast<const f32x4 *>(lds + w * VBUF + (wave * MD + d) * 1024 + lane * 16) * f;
        }
        const uint32_t r = (rb * QT + t) * 16 + r16;
        if (r >= R) continue;
        if (a.part) {
            const size_t at_row = ((size_t)split * a.nkv + g) * R + r;
            float *w = a.part + at_row * HD, *mlp = a.part + (size_t)a.splits * a.nkv * R * HD + 2 * at_row;
#pragma unroll
            for (int d = 0; d < MD; ++d) *reinterpret_cast<f32x4 *>(w + 16 * (wave * MD + d) + 4 * q4) = x[d];
            if (wave == 0 && q4 == 0) mlp[0] = top, mlp[1] = all;
        } else {
            const bool any = all != 0.0f || sees_any(a, tok[t]);
            uint16_t *out = a.out + ((size_t)tok[t] * a.nh + g * per + r % per) * a.hd;
#pragma unroll
            for (int d = 0; d < MD; ++d) {
                const uint32_t dim = 16 * (wave * MD + d) + 4 * q4;
                if (dim < a.hd) *reinterpret_cast<u32x2 *>(out + dim) = finish(x[d], all, any);
            }
        }
    }
}

// Merges the splits' (o, m, l): a thread takes four dimensions of a query row, GR threads its
// splits in turn.
template <int HD, int GR>
__global__ __launch_bounds__(256) void attention_mxfp4_merge(const MxAttn a) {
    constexpr uint32_t QUADS = HD / 4, PER = 256 / (QUADS * GR);   // rows of a workgroup
    static_assert(PER >= 1, "rows");
    __shared__ float lds[GR > 1 ? 6 * 256 : 1];
    const uint32_t quad = threadIdx.x % QUADS, grp = threadIdx.x / QUADS % GR;
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, all_rows = a.nkv * R;
    const uint32_t at = blockIdx.x * PER + threadIdx.x / (QUADS * GR), row = min(at, all_rows - 1);
    const float *w = a.part + (size_t)row * HD + 4 * quad, *mlp = a.part + (size_t)a.splits * all_rows * HD + 2 * (size_t)row;
    const size_t step = (size_t)all_rows * HD, step_ml = 2 * (size_t)all_rows;
    float top = -INFINITY, l = 0.0f;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (uint32_t s = grp; s < a.splits; s += GR) top = fmaxf(top, mlp[s * step_ml]);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll 8
    for (uint32_t s = grp; s < a.splits; s += GR) {
        const float f = exp2f(mlp[s * step_ml] - ref);
        l += mlp[s * step_ml + 1] * f;
        o += *reinterpret_cast<const f32x4 *>(w + s * step) * f;
    }
    if constexpr (GR > 1) {
        float *mine = lds + threadIdx.x;
        mine[0] = top, mine[256] = l;
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[512 + 256 * e] = o[e];
        __syncthreads();
        if (grp > 0) return;
        const float *p = lds + threadIdx.x;
#pragma unroll
        for (int k = 1; k < GR; ++k) top = fmaxf(top, p[k * QUADS]);
        const float base = top == -INFINITY ? 0.0f : top;
        l = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < GR; ++k) {
            const float f = exp2f(p[k * QUADS] - base);
            l += p[k * QUADS + 256] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += p[k * QUADS + 512 + 256 * e] * f;
        }
    }
    if (at >= all_rows || 4 * quad >= a.hd) return;
    const uint32_t g = row / R, r = row % R, tok = r / per;
    const bool any = l != 0.0f || sees_any(a, tok);
    *reinterpret_cast<u32x2 *>(a.out + ((size_t)tok * a.nh + g * per + r % per) * a.hd + 4 * quad) = finish(o, l, any);
}

template <int HD, int QT>
int launch(const MxAttn &a, hipStream_t st) {
    constexpr int LDS = MXA_WAVES * MXA_TILE * 2 * HD;
    static_assert(LDS <= 160 * 1024, "LDS");
    const unsigned grid = (a.units + MXA_XCDS - 1) / MXA_XCDS * MXA_XCDS * a.row_blocks;
    hipLaunchKernelGGL((attention_mxfp4<HD, QT>), dim3(grid), dim3(64 * MXA_WAVES), LDS, st, a);
    if (int rc = check_launch("attention_mxfp4")) return rc;
    if (a.splits < 2) return RENG_HIP_OK;
    const uint32_t rows = a.tokens * a.nh;
    constexpr int GR = 256 / (HD / 4);
    if (a.splits >= 8)
        hipLaunchKernelGGL((attention_mxfp4_merge<HD, GR>), dim3(rows), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((attention_mxfp4_merge<HD, 1>), dim3((rows + GR - 1) / GR), dim3(256), 0, st, a);
    return check_launch("attention_mxfp4_merge");
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API size_t reng_hip_attention_mxfp4_workspace_bytes(size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                                             size_t len, size_t tokens) {
    if (n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads || n_heads > 4096 || head_dim > 256) return 0;
    if (tokens > RENG_HIP_TREE_MAX_TOKENS) tokens = RENG_HIP_TREE_MAX_TOKENS;
    if (len > RENG_HIP_ATTENTION_MAX_LEN) len = RENG_HIP_ATTENTION_MAX_LEN;
    return mxa_workspace(n_heads, n_kv_heads, head_dim, len, tokens);
}

RENG_HIP_API int reng_hip_attention_mxfp4(const uint16_t *q, const reng_hip_mx_cache *cache, size_t n_heads, size_t len,
                                          size_t tokens, const uint32_t *mask, float scale, void *workspace,
                                          size_t workspace_bytes, uint16_t *out, void *stream) {
    clear_error();
    if (int rc = check_mx_cache(cache)) return rc;
    const reng_hip_mx_cache &c = *cache;
    RENG_REQUIRE(n_heads > 0 && n_heads % c.n_kv_heads == 0, "%zu query heads are not a multiple of %zu key/value heads",
                 n_heads, c.n_kv_heads);
    RENG_REQUIRE(n_heads <= 4096, "%zu query heads; at most 4096", n_heads);
    RENG_REQUIRE(tokens >= 1 && tokens <= RENG_HIP_TREE_MAX_TOKENS, "%zu tokens; expected 1 to %d", tokens,
                 RENG_HIP_TREE_MAX_TOKENS);
    RENG_REQUIRE(len <= RENG_HIP_ATTENTION_MAX_LEN && len + tokens <= RENG_HIP_ATTENTION_MAX_LEN,
                 "%zu context rows and %zu tokens; at most %d rows", len, tokens, RENG_HIP_ATTENTION_MAX_LEN);
    RENG_REQUIRE(len + tokens <= c.capacity, "%zu context rows and %zu tokens in a cache of %zu", len, tokens, c.capacity);
    RENG_REQUIRE(scale - scale == 0.0f, "scale is not finite");
    RENG_REQUIRE(q && out, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(mask) & 3) == 0,
                 "q and out must be 16-byte aligned, mask 4-byte");
    const MxAttnPlan p = mxa_plan(n_heads, c.n_kv_heads, c.head_dim, len, tokens, (size_t)device_props().cus);
    const size_t need = mxa_workspace(n_heads, c.n_kv_heads, c.head_dim, len, tokens);
    RENG_REQUIRE(workspace_bytes >= need, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    RENG_REQUIRE(need == 0 || workspace, "null workspace");
    RENG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "workspace must be 16-byte aligned");
    const MxAttn a{q,
                   c.k_codes,
                   c.k_scales,
                   c.v_codes,
                   c.v_scales,
                   c.capacity,
                   (uint32_t)n_heads,
                   (uint32_t)c.n_kv_heads,
                   (uint32_t)c.head_dim,
                   (uint32_t)scale_pitch(c.head_dim),
                   (uint32_t)len,
                   (uint32_t)tokens,
                   mask,
                   (uint32_t)((tokens + 31) / 32),
                   scale,
                   out,
                   p.row_blocks,
                   (uint32_t)(p.splits * c.n_kv_heads),
                   p.splits,
                   p.tiles / p.splits,
                   p.tiles % p.splits,
                   p.splits > 1 ? static_cast<float *>(workspace) : nullptr};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p.hdp == 256) return p.qt == 1 ? launch<256, 1>(a, st) : launch<256, 2>(a, st);
    if (p.hdp == 128) return p.qt == 1 ? launch<128, 1>(a, st) : p.qt == 2 ? launch<128, 2>(a, st) : launch<128, 4>(a, st);
    return p.qt == 1 ? launch<64, 1>(a, st) : p.qt == 2 ? launch<64, 2>(a, st) : launch<64, 4>(a, st);
}
