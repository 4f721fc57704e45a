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
// that share it) go 16 to a wave, eight waves taking tiles of 32 cache rows of their own in
// turn, or, where there are many, 32 to a wave over tiles that a workgroup shares in LDS.
// Splits of the cache merge in a second kernel (mx_attention_plan.h).
//
// Few rows: per tile a wave forms S^T = K Q^T on v_mfma_f32_16x16x32_bf16. Lane l has key l % 16 and,
// of its dimensions, the quarter l / 16: the order in which dimensions are summed is free, so
// a lane's codes are consecutive bytes and lie under one scale (two of 256 dimensions), and the
// queries' registers follow that order. The results have query l % 16 and four keys from
// 4 (l / 16), which is how O^T = V^T P^T takes the weights. V^T comes from LDS, where a
// wave puts a tile's values as bf16, by transposing reads.
//
// A row whose key or value holds a scale from 253 on (NaN, or magnitudes bf16 ends at)
// counts as NaN: its key's scale becomes NaN and its value's 1, so that its score decides
// who meets it, and a weight of 0 takes nothing from a value.
//
// Weights meet their values as bf16, the matrix cores' type (a second product for what bf16 leaves takes
// one token after 131071 rows from 31.4 to 33.2 us, and half as many products more where they bound it), and are
// summed as they were: so an output is off by at most 2^-8 sum p |v|. A sum of the rounded ones takes back
// a dominant weight's rounding where its value dominates too (2-norm 0.0019 for 0.0023 with a few rows that
// matter), but adds it where that value is 0, which doubles the bound.
//
// What bounds it: one token after 32768 rows (32 heads on 8, 36 MB of cache) 14.7 us, 11.6 of
// them the rows' kernel and 3.7 the merge: two launches and the start of each; after 131071 31.5.
// A chain of 1024 after 16384 (40 on 8) 349 us, 1.0 PFLOP/s: the matrix cores and, in turn with them,
// the exponentials; after none 45.8, masked steps without turns.
#include <float.h>

#include <type_traits>

#include "common.h"
#include "mfma_pipe.h"
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
typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// All arguments asked for at once: left to itself the compiler reads them where they are used, and waits for one
// cache line of them after the other (one token after 4096 rows 9.3 us, and 9.1 so).
__device__ __forceinline__ void arguments(const MxAttn &a) {
    asm volatile("" ::"s"(a.q), "s"(a.kc), "s"(a.ks), "s"(a.vc), "s"(a.vs), "s"(a.cap), "s"(a.nh), "s"(a.nkv), "s"(a.hd),
                 "s"(a.sp), "s"(a.len), "s"(a.tokens), "s"(a.mask), "s"(a.words), "s"(a.scale), "s"(a.out),
                 "s"(a.row_blocks), "s"(a.units), "s"(a.splits), "s"(a.base), "s"(a.more), "s"(a.part));
}

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

// The rows of a head as a buffer: what lies behind them reads as zeros. (A scalar offset would not
// count in that: the whole offset is the lane's.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint8_t *p, size_t head, uint32_t rows, uint32_t pitch) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p) + head * pitch, 0, rows * pitch, 0x00020000);
}
constexpr uint32_t NOTHING = 0x7fffffffu;   // past every buffer

// The queries of key/value head g as a buffer, and eight dimensions of one, `row` heads on from the first.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t queries_of(const MxAttn &a, uint32_t g) {
    const uint32_t per = a.nh / a.nkv, before = g * per * a.hd * 2;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(a.q) + before / 2, 0, a.tokens * a.nh * a.hd * 2 - before,
                                             0x00020000);
}
__device__ __forceinline__ u32x4 query_chunk(const __amdgpu_buffer_rsrc_t &rq, const MxAttn &a, uint32_t row, uint32_t dim) {
    const uint32_t at = dim < a.hd ? (row * a.hd + dim) * 2 : 0xfffffff0u;   // up to 2^31 bytes of queries
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, at, 0, 0));
}

// The slot of 16-byte chunk c of a tile's row r. Eight consecutive rows written at one chunk
// and four read over two chunks lie in different slots.
__device__ __forceinline__ uint32_t value_slot(uint32_t r, uint32_t c) {
    return c ^ (((r & 3) << 1) | ((r >> 2) & 1));
}

// ------------------------------------------------------------ few query rows
//
// NW waves, each with the same 16 query rows and tiles of its own, whose codes are on the
// way while the one before is worked on. One token after 32768: two and four tiles ahead 18.3 and
// 19.9 us where one takes 17.5; four and sixteen waves 19.2 and 19.3 where eight take 17.5.
template <int HD, int NW>
__global__ __launch_bounds__(64 * NW) void attention_mxfp4(const MxAttn a) {
    constexpr int ST = HD / 32, DT = HD / 16;   // products a score; tiles of dimensions
    constexpr int LB = HD / 8, CH = LB <= 16 ? 1 : LB / 16;     // bytes of a lane; 16-byte chunks of them
    constexpr int ROWB = 2 * HD, VBUF = MXA_TILE * ROWB;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float ml[2][NW][16];
    // Workgroups go to the XCDs in turn: the row blocks of one split and key/value head
    // follow each other on one XCD, whose L2 gives them the rows after the first.
    arguments(a);
    const uint32_t b = blockIdx.x / MXA_XCDS, rb = b % a.row_blocks;
    const uint32_t unit = b / a.row_blocks * MXA_XCDS + blockIdx.x % MXA_XCDS;
    if (unit >= a.units) return;
    const uint32_t g = unit % a.nkv, split = unit / a.nkv;
    const uint32_t lane = threadIdx.x & 63, r16 = lane & 15, q4 = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, rows = a.len + a.tokens;
    uint8_t *vbuf = lds + wave * VBUF;

    // This lane's query row (clamped: rows past the last are not stored).
    // scale < 0 goes into the queries' signs, so that the largest product is the largest score.
    const float c = fabsf(a.scale) * 1.44269504088896341f;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    const uint32_t dim0 = q4 * (HD / 4);   // this lane's dimensions
    const uint32_t r0 = rb * 16 + r16, r = min(r0, R - 1), tok = r / per;
    const size_t qrow = (size_t)tok * a.nh + g * per + r % per;
    u32x4 qw[ST];
    const __amdgpu_buffer_rsrc_t rq = queries_of(a, g);
#pragma unroll
    for (int e = 0; e < ST; ++e) qw[e] = query_chunk(rq, a, tok * a.nh + r % per, dim0 + 8 * e);

    // The split's tiles, cut for a chain at the last row its tokens see.
    const uint32_t t0 = split * a.base + min(split, a.more);
    uint32_t t1 = t0 + a.base + (split < a.more);
    if (!a.mask) {
        const uint32_t last = min(rb * 16 + 15, R - 1) / per;
        t1 = min(t1, (a.len + last) / MXA_TILE + 1);
    }

    const size_t head = (size_t)g * a.cap;
    const uint32_t rowb = a.hd / 2;
    struct Codes {
        uint32_t w[LB / 4];
        uint32_t s[CH];   // scale bytes
    };
    // Where this lane's codes of a row lie, chunk by chunk; zeros past the head's dimensions.
    uint32_t at_codes[CH], at_scale[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const bool on = dim0 + 32 * i < a.hd;
        at_codes[i] = on ? r16 * rowb + dim0 / 2 + 16 * i : NOTHING;
        at_scale[i] = on ? r16 * a.sp + dim0 / 32 + i : NOTHING;
    }
    Codes kn[2], vn[2];   // the next tile's: keys 16 u + l % 16
    const __amdgpu_buffer_rsrc_t rkc = rows_of(a.kc, head, rows, rowb), rks = rows_of(a.ks, head, rows, a.sp);
    const __amdgpu_buffer_rsrc_t rvc = rows_of(a.vc, head, rows, rowb), rvs = rows_of(a.vs, head, rows, a.sp);
    auto fetch = [&](uint32_t tile) __attribute__((always_inline)) {
        auto load = [&](Codes &v, const __amdgpu_buffer_rsrc_t &rc, const __amdgpu_buffer_rsrc_t &rs,
                        uint32_t j) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                v.s[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs, at_scale[i] + j * a.sp, 0, 0);
                if constexpr (LB == 8) {
                    const u32x2 x =
                        __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rc, at_codes[i] + j * rowb, 0, 0));
                    v.w[0] = x.x, v.w[1] = x.y;
                } else {
                    const u32x4 x =
                        __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, at_codes[i] + j * rowb, 0, 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v.w[4 * i + e] = x[e];
                }
            }
        };
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            load(kn[u], rkc, rks, tile * MXA_TILE + 16 * u);
            load(vn[u], rvc, rvs, tile * MXA_TILE + 16 * u);
        }
    };

    f32x4 o[DT];
    float m = -INFINITY, l = 0.0f;   // the running maximum of the products, this lane's share of the sum
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0, 0, 0, 0};
    fetch(t0 + wave);   // behind the queries' loads, before anything waits for them
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 qf[ST];
#pragma unroll
    for (int e = 0; e < ST; ++e) qf[e] = __builtin_bit_cast(bf16x8, qw[e] ^ flip);
    for (uint32_t tile = t0 + wave; tile < t1; tile += NW) {
        const uint32_t j0 = tile * MXA_TILE;
        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {   // keys 16 u ..
            Codes k = kn[u], v = vn[u];
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
            s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < ST; ++e) {
                const bf16x8 kf = __builtin_bit_cast(bf16x8, decode8(k.w[e], scale_operand(k.s[e * CH / ST])));
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[e], s[u], 0, 0, 0);
            }
        }
        if (tile + NW < t1) fetch(tile + NW);
        asm volatile("" ::: "memory");   // the values are read by other lanes than wrote them, in the wave's own order
        const bool masked = j0 + MXA_TILE > a.len;
        uint32_t see = 0xffffffffu;
        if (masked) {
            see = seen_bits(a, tok, j0) >> (4 * q4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!((see >> (16 * (i / 4) + i % 4)) & 1)) s[i / 4][i % 4] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        // The maximum moves, and what is summed so far is scaled down, only where a
        // score passes it by more than 2^8: weights up to 256 lose nothing in f32 or bf16.
        if (__builtin_amdgcn_ballot_w64((mx - m) * c > 8.0f || (m == -INFINITY && mx > m))) {
            mx = query_max(mx);
            const bool move = (mx - m) * c > 8.0f || (m == -INFINITY && mx > m);
            const float f = !move ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * c);
            if (move) m = mx;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
        // Against the lowest value where the maximum has none or, in base 2, lies below f32: exponentials of 0 then.
        const float mc = fmaxf(m * c, -FLT_MAX);
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], c, -mc));
            if (masked) p[i] = (see >> (16 * (i / 4) + i % 4)) & 1 ? p[i] : 0.0f;
            l += p[i];
        }
        const bf16x8 pw = __builtin_bit_cast(bf16x8, u32x4{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]),
                                                           pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7])});
        // V^T of the tile's rows in the order of the weights. Lane: dimensions 4 (l % 4) .. + 3 of a row.
        const uint32_t row = 4 * q4 + r16 / 4;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const uint32_t ch = 2 * d + (r16 & 3) / 2, in = 8 * (r16 & 1);
            const u32x2 v0 = read_tr(vbuf + row * ROWB + 16 * value_slot(row, ch) + in);
            const u32x2 v1 = read_tr(vbuf + (row + 16) * ROWB + 16 * value_slot(row + 16, ch) + in);
            const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{v0.x, v0.y, v1.x, v1.y});
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pw, o[d], 0, 0, 0);
        }
        asm volatile("" ::: "memory");
    }

    // The waves' (o, m, l) through LDS, the dimensions' tiles merged by the waves in turn.
    constexpr int MD = (DT + NW - 1) / NW;
    __syncthreads();
    const float sum = query_sum(l), top_c = m == -INFINITY ? -INFINITY : m * c;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(vbuf + d * 1024 + lane * 16) = o[d];
    if (q4 == 0) ml[0][wave][r16] = top_c, ml[1][wave][r16] = sum;
    __syncthreads();
    float top = ml[0][0][r16];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, ml[0][w][r16]);
    const float at = top == -INFINITY ? 0.0f : top;
    float all = 0.0f;
    f32x4 x[MD];
#pragma unroll
    for (int i = 0; i < MD; ++i) x[i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml[0][w][r16] - at);
        all += ml[1][w][r16] * f;
#pragma unroll
        for (int i = 0; i < MD; ++i)
            x[i] += *reinterpret_cast<const f32x4 *>(lds + w * VBUF + (wave + i * NW) % DT * 1024 + lane * 16) * f;
    }
    if (r0 >= R) return;
    const size_t at_row = ((size_t)split * a.nkv + g) * R + r0;
    const bool any = a.part || all != 0.0f || sees_any(a, tok);
    if (a.part && wave == 0 && q4 == 0) {
        float *mlp = a.part + (size_t)a.splits * a.nkv * R * HD + 2 * at_row;
        mlp[0] = top, mlp[1] = all;
    }
#pragma unroll
    for (int i = 0; i < MD; ++i) {
        const uint32_t d = wave + i * NW, dim = 16 * d + 4 * q4;
        if (d >= DT) break;
        if (a.part) *reinterpret_cast<f32x4 *>(a.part + at_row * HD + dim) = x[i];
        else if (dim < a.hd) *reinterpret_cast<u32x2 *>(a.out + qrow * a.hd + dim) = finish(x[i], all, any);
    }
}

// ------------------------------------------------------------ many query rows
//
// The query rows go 32 to a wave. A workgroup's RW waves of a key group share its tiles of TK
// cache rows, which they bring into LDS as bf16: a wave reads its share of a later tile's codes into
// registers and writes their values a step after. KW key groups take tiles in turn and merge
// in LDS. Products are v_mfma_f32_32x32x16_bf16: S^T = K Q^T leaves a lane 16 scores of one query per
// 32 keys, in the order in which O^T = V^T P^T takes the weights.
template <int HD, int RW, int KW, int TK, int S>
struct MxShape {
    static constexpr int W = RW * KW, P2 = HD / 8, ROWB = 2 * HD;   // 16-byte chunks and bytes of a row
    static constexpr int TILE = TK * ROWB, STAGE = 2 * TILE;        // keys then values
    static constexpr int NB = HD / 32, RT = 64 / NB;                // blocks of a row; rows of a wave's part
    static constexpr int PARTS = 2 * TK / RT, MINE = (PARTS + RW - 1) / RW;   // parts of a tile; of a wave
    static constexpr int PW = HD * 32 + 128;                        // floats that a wave merges
    static constexpr int RING = KW * S * STAGE, MERGE = (KW - 1) * RW * PW * 4, LDS = RING > MERGE ? RING : MERGE;
    static constexpr int DB = HD / 32, KB = TK / 32;
    static constexpr int AHEAD = 6;                                 // products whose operands are read ahead
    static constexpr bool TURNS = RW == 8;                          // the waves' halves take turns
    static_assert(!TURNS || (KW == 1 && S == 4), "one wave of each half on a SIMD, four slots");
    static_assert(TURNS || S == 2, "a tile is written while the one before it is used");
    static_assert(LDS <= 160 * 1024, "LDS");
};

// 32 rows are read at one chunk, eight consecutive ones are written at one.
__device__ __forceinline__ uint32_t key_slot(uint32_t r, uint32_t c) { return c ^ (r & 7); }

__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int HD, int RW, int KW, int TK, int S>
__global__ __launch_bounds__(64 * RW * KW) void attention_mxfp4_tiles(const MxAttn a) {
    using T = MxShape<HD, RW, KW, TK, S>;
    constexpr int ROWB = T::ROWB, DB = T::DB, KB = T::KB, AHEAD = T::AHEAD, MINE = T::MINE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    arguments(a);
    const uint32_t b = blockIdx.x / MXA_XCDS, rb = b % a.row_blocks;
    const uint32_t unit = b / a.row_blocks * MXA_XCDS + blockIdx.x % MXA_XCDS;
    if (unit >= a.units) return;
    const uint32_t g = unit % a.nkv, split = unit / a.nkv;
    const uint32_t lane = threadIdx.x & 63, h = lane >> 5, ql = lane & 31;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW, kg = wave / RW;
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, rows = a.len + a.tokens;

    // This lane's query row (clamped: rows past the last are not stored).
    const uint32_t r0 = (rb * RW + rw) * 32 + ql, r = min(r0, R - 1), tok = r / per;
    const size_t qrow = (size_t)tok * a.nh + g * per + r % per;
    const float c = fabsf(a.scale) * 1.44269504088896341f;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    u32x4 qw[HD / 16];
    const __amdgpu_buffer_rsrc_t rq = queries_of(a, g);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) qw[s] = query_chunk(rq, a, tok * a.nh + r % per, 16 * s + 8 * h);

    // The split's tiles, cut for a chain at the last row its tokens see.
    const uint32_t t0 = split * a.base + min(split, a.more);
    uint32_t t1 = t0 + a.base + (split < a.more);
    if (!a.mask) {
        const uint32_t last = min((rb * RW + RW) * 32 - 1, R - 1) / per;
        t1 = min(t1, (a.len + last) / TK + 1);
    }
    const uint32_t n = t1 > t0 ? t1 - t0 : 0, steps = (n + KW - 1) / KW;
    auto has = [&](uint32_t step) { return step * KW + kg < n; };
    auto tile_row = [&](uint32_t step) { return (t0 + step * KW + kg) * TK; };
    uint8_t *ring = lds + kg * (S * T::STAGE);
    auto keys = [&](uint32_t step) { return ring + (step % S) * T::STAGE; };

    // A part is 64 blocks of 32 codes: a block a lane, RT rows of keys (the first half of the parts)
    // or values. fetch() reads this wave's parts of a tile, put() writes their values.
    const size_t head = (size_t)g * a.cap;
    const uint32_t prow = lane % T::RT, blk = lane / T::RT, rowb = a.hd / 2;
    const uint32_t at_codes = 32 * blk < a.hd ? prow * rowb + 16 * blk : NOTHING;
    const uint32_t at_scale = 32 * blk < a.hd ? prow * a.sp + blk : NOTHING;
    u32x4 codes[MINE];
    uint32_t byte[MINE], other[MINE];   // the block's scale; for a key its value's, too
    __amdgpu_buffer_rsrc_t rc[MINE], rs[MINE];
    const __amdgpu_buffer_rsrc_t rvs = rows_of(a.vs, head, rows, a.sp);
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const bool values = rw + i * RW >= T::PARTS / 2;
        rc[i] = rows_of(values ? a.vc : a.kc, head, rows, rowb);
        rs[i] = rows_of(values ? a.vs : a.ks, head, rows, a.sp);
    }
    auto fetch = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const uint32_t part = rw + i * RW;
            if (part >= T::PARTS) break;
            const uint32_t j = tile_row(step) + part % (T::PARTS / 2) * T::RT;
            codes[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rc[i], at_codes + j * rowb, 0, 0));
            byte[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs[i], at_scale + j * a.sp, 0, 0);
            other[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rvs, at_scale + j * a.sp, 0, 0);
        }
    };
    auto put = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const uint32_t part = rw + i * RW, half = T::PARTS / 2;
            if (part >= T::PARTS) break;
            const bool values = part >= half;
            const uint32_t row = (values ? part - half : part) * T::RT + prow;
            const bool odd = max(byte[i], other[i]) >= 253;
            const float s = scale_operand(odd ? (values ? ONE_BYTE : NAN_BYTE) : byte[i]);
            uint8_t *to = keys(step) + (values ? T::TILE : 0) + row * ROWB;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t ch = 4 * blk + e;
                *reinterpret_cast<u32x4 *>(to + 16 * (values ? value_slot(row, ch) : key_slot(row, ch))) = decode8(codes[i][e], s);
            }
        }
    };

    fetch(0);   // behind the queries' loads, before anything waits for them
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 qf[HD / 16];
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) qf[e] = __builtin_bit_cast(bf16x8, qw[e] ^ flip);

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;   // the running maximum of the products, this lane's share of the sum
    f32x16 s[KB];                    // a tile's scores, before the scale
    u32x4 pw[2 * KB];                // its weights in bf16: the 16 rows 16 u .. of each 32 as PV takes them

    // 16 dimensions of 32 of a tile's keys as the matrix cores take them.
    auto key_frag = [&](const uint8_t *ks, int kb, int st) __attribute__((always_inline)) {
        const uint32_t row = 32 * kb + ql;
        return *reinterpret_cast<const u32x4 *>(ks + row * ROWB + key_slot(row, 2 * st + h) * 16);
    };
    const f32x16 zero = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f,
                         0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    auto weights = [&](auto masked_c, uint32_t j0) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_c)::value;
        uint32_t see[KB];   // bit 8 (i / 4) + i % 4: whether score i counts
        if constexpr (MASKED) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                see[kb] = seen_bits(a, tok, j0 + 32 * kb) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!((see[kb] >> (8 * (i / 4) + i % 4)) & 1)) s[kb][i] = -INFINITY;
            }
        }
        // Four chains each for the maximum and the sum: one would wait for every step's result.
        float mx4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx4[i] = s[0][i];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = kb ? 0 : 4; i < 16; i += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mx4[e] = i + 4 < 16 ? fmaxf(fmaxf(mx4[e], s[kb][i + e]), s[kb][i + 4 + e]) : fmaxf(mx4[e], s[kb][i + e]);
        const float mx = both_max(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
        // The maximum moves, and what is summed so far is scaled down, only where a
        // score passes it by more than 2^8: weights up to 256 lose nothing in f32 or bf16.
        const bool move = (mx - m) * c > 8.0f || (m == -INFINITY && mx > m);
        if (__builtin_amdgcn_ballot_w64(move)) {
            const float f = !move ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * c);
            if (move) m = mx;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
        }
        // Against the lowest value where the maximum has none or, in base 2, lies below f32: exponentials of 0 then.
        const float mc = fmaxf(m * c, -FLT_MAX);
        float l4[4] = {l, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = 8 * u + i;
                    p[i] = __builtin_amdgcn_exp2f(fmaf(s[kb][k], c, -mc));
                    if constexpr (MASKED) p[i] = (see[kb] >> (8 * (k / 4) + k % 4)) & 1 ? p[i] : 0.0f;
                    l4[i % 4] += p[i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) pw[2 * kb + u][i] = pack_bf16(p[2 * i], p[2 * i + 1]);
            }
        l = (l4[0] + l4[1]) + (l4[2] + l4[3]);
        // Formed here, not where they are used: that may be behind a barrier.
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i) asm volatile("" : "+v"(pw[i]));
    };
    // V^T of the 16 rows from 32 kb + 16 u as the matrix cores take it. Lane: dimensions
    // 4 (l % 4) .. + 3 of a row, from the 16 at 32 d + 16 (l / 16 % 2).
    auto value_frag = [&](const uint8_t *vs, int kb, int u, int d) __attribute__((always_inline)) {
        const uint32_t row = 32 * kb + 16 * u + 4 * h + (lane & 15) / 4;
        const uint32_t dim = 32 * d + (lane & 16) + 4 * (lane & 3), in = 2 * (dim & 7), ch = dim / 8;
        const u32x2 v0 = read_tr(vs + row * ROWB + value_slot(row, ch) * 16 + in);
        const u32x2 v1 = read_tr(vs + (row + 8) * ROWB + value_slot(row + 8, ch) * 16 + in);
        return u32x4{v0.x, v0.y, v1.x, v1.y};
    };
    // A run of matrix products in the order written, each one's operand read from LDS AHEAD
    // products before it is used: the values of a tile (VALUES) and the scores of another.
    auto run = [&](auto values_c, auto scores_c, const uint8_t *vs, const uint8_t *ks) __attribute__((always_inline)) {
        constexpr int NV = decltype(values_c)::value ? 2 * KB * DB : 0, NK = decltype(scores_c)::value ? KB * HD / 16 : 0;
        constexpr int N = NV + NK;
        auto read = [&](int p) __attribute__((always_inline)) {
            return p < NV ? value_frag(vs, p / DB / 2, p / DB % 2, p % DB) : key_frag(ks, (p - NV) % KB, (p - NV) / KB);
        };
        u32x4 f[AHEAD];
#pragma unroll
        for (int p = 0; p < AHEAD && p < N; ++p) f[p] = read(p);
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const bf16x8 x = __builtin_bit_cast(bf16x8, f[p % AHEAD]);
            if (p < NV) {
                o[p % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, __builtin_bit_cast(bf16x8, pw[p / DB]), o[p % DB],
                                                                    0, 0, 0);
            } else {
                const int kb = (p - NV) % KB, st = (p - NV) / KB;
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, qf[st], st ? s[kb] : zero, 0, 0, 0);
            }
            if (p + AHEAD < N) f[p % AHEAD] = read(p + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const std::true_type yes{};
    const std::false_type no{};
    // Every LDS access of this wave is done before another wave reads or writes there.
    auto barrier = [&] {
        pipe::wait_lgkm0();
        pipe::lds_barrier();
    };
    // The first `whole` steps' tiles lie within the context; the others look at the mask, in
    // a loop of their own, whose registers the first does not pay for.
    const uint32_t in = min(n, max(a.len / TK, t0) - t0), whole = in / KW;
    auto masked_step = [&](uint32_t step, uint32_t next) __attribute__((always_inline)) {
        barrier();   // the tile is written, and every wave is done with the slot before
        if (has(next)) {
            put(next);
            fetch(next + 1);
        }
        if (!has(step)) return;
        run(no, yes, nullptr, keys(step));
        weights(yes, tile_row(step));
        run(yes, no, keys(step) + T::TILE, nullptr);
    };
    if constexpr (T::TURNS) {
        // The waves' two halves, one of each on a SIMD, take turns: while one half runs its
        // matrix products (a tile's values, the next tile's scores), the other half's weights and
        // its share of a later tile use the vector unit. A phase ends at a barrier; the
        // second half runs one phase behind. Tile i's scores are formed in phases 2 i and 2 i + 1
        // and its values used in phases 2 i + 2 and 2 i + 3, so with four slots the first half
        // may write tile i + 2 in phase 2 i + 1, the second tile i + 3 in phase 2 i + 2.
        const bool second = wave >= T::W / 2;
        const uint32_t far = second ? 3 : 2;
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i)
            if (i < far && has(i)) {
                put(i);
                fetch(i + 1);
            }
        if (whole) {
            barrier();
            if (second) barrier();
            run(no, yes, nullptr, keys(0));
            for (uint32_t i = 0; i < whole; ++i) {
                barrier();
                if (has(i + far)) {
                    put(i + far);
                    fetch(i + far + 1);
                }
                weights(no, 0);
                barrier();
                // Behind the last tile these scores are not used.
                run(yes, yes, keys(i) + T::TILE, keys(i + 1));
            }
            if (!second) barrier();
        }
        for (uint32_t i = whole; i < steps; ++i) masked_step(i, i + far);
    } else {
        if (has(0)) {
            put(0);
            fetch(1);
        }
        uint32_t step = 0;
        for (; step < whole; ++step) {
            barrier();
            if (has(step + 1)) {
                put(step + 1);
                fetch(step + 2);
            }
            run(no, yes, nullptr, keys(step));
            weights(no, 0);
            run(yes, no, keys(step) + T::TILE, nullptr);
        }
        for (; step < steps; ++step) masked_step(step, step + 1);
    }
    l = both_sum(l);
    float mc = m == -INFINITY ? -INFINITY : m * c;

    if constexpr (KW > 1) {
        // The other key groups' (o, m, l) through LDS, lane by lane.
        __syncthreads();
        float *buf = reinterpret_cast<float *>(lds);
        constexpr int PW = T::PW;
        if (kg > 0) {
            float *w = buf + ((kg - 1) * RW + rw) * PW;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4 *>(w + (d * 4 + i) * 256 + lane * 4) =
                        f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            w[DB * 1024 + lane] = mc;
            w[DB * 1024 + 64 + lane] = l;
        }
        __syncthreads();
        if (kg > 0) return;
        float top = mc;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) top = fmaxf(top, buf[(k * RW + rw) * PW + DB * 1024 + lane]);
        const float at = top == -INFINITY ? 0.0f : top;
        float f = __builtin_amdgcn_exp2f(mc - at);
        l *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= f;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) {
            const float *w = buf + (k * RW + rw) * PW;
            f = __builtin_amdgcn_exp2f(w[DB * 1024 + lane] - at);
            l += w[DB * 1024 + 64 + lane] * f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(w + (d * 4 + i) * 256 + lane * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][4 * i + e] += v[e] * f;
                }
        }
        mc = top;
    }
    if (r0 >= R) return;
    // A lane has dimensions 32 d + 8 i + 4 h .. + 3 of its row.
    if (a.part) {
        const size_t at_row = ((size_t)split * a.nkv + g) * R + r0;
        float *w = a.part + at_row * HD, *mlp = a.part + (size_t)a.splits * a.nkv * R * HD + 2 * at_row;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4 *>(w + 32 * d + 8 * i + 4 * h) =
                    f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (h == 0) mlp[0] = mc, mlp[1] = l;
        return;
    }
    const bool any = l != 0.0f || sees_any(a, tok);
    uint16_t *out = a.out + qrow * a.hd;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t dim = 32 * d + 8 * i + 4 * h;
            if (dim < a.hd)
                *reinterpret_cast<u32x2 *>(out + dim) =
                    finish(f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}, l, any);
        }
}

// Merges the splits' (o, m, l): a thread takes four dimensions of a query row and up to sixteen splits, all of
// which it asks for at once; GR threads share a row's splits and meet in LDS. Latency is the time: with 4, 8 and
// 32 splits a thread one token after 32768 rows took 16.0, 17.0 and 16.8 us, with 16 15.7.
constexpr uint32_t MERGE_SPLITS = 16;
static_assert(MXA_SPLIT_MAX <= 4 * MERGE_SPLITS, "four threads a row hold all splits");

template <int HD, int GR>
__global__ __launch_bounds__(GR > 1 ? HD / 4 * GR : 256) void attention_mxfp4_merge(const MxAttn a) {
    constexpr uint32_t T = GR > 1 ? HD / 4 * GR : 256, QUADS = HD / 4, PER = T / (QUADS * GR);   // threads, rows of a workgroup
    __shared__ float lds[GR > 1 ? 6 * T : 1];
    arguments(a);
    const uint32_t quad = threadIdx.x % QUADS, grp = threadIdx.x / QUADS % GR;
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, all_rows = a.nkv * R;
    const uint32_t at = blockIdx.x * PER + threadIdx.x / (QUADS * GR), row = min(at, all_rows - 1);
    const float *w = a.part + (size_t)row * HD + 4 * quad, *mlp = a.part + (size_t)a.splits * all_rows * HD + 2 * (size_t)row;
    const size_t step = (size_t)all_rows * HD, step_ml = 2 * (size_t)all_rows;
    float ms[MERGE_SPLITS], ls[MERGE_SPLITS];
    f32x4 os[MERGE_SPLITS];
#pragma unroll
    for (uint32_t i = 0; i < MERGE_SPLITS; ++i) {
        const uint32_t s = grp + i * GR;
        ms[i] = -INFINITY, ls[i] = 0.0f, os[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (s < a.splits) {
            const float2 v = *reinterpret_cast<const float2 *>(mlp + s * step_ml);
            ms[i] = v.x, ls[i] = v.y;
            os[i] = *reinterpret_cast<const f32x4 *>(w + s * step);
        }
    }
    float top = -INFINITY, l = 0.0f;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < MERGE_SPLITS; ++i) top = fmaxf(top, ms[i]);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (uint32_t i = 0; i < MERGE_SPLITS; ++i) {
        const float f = __builtin_amdgcn_exp2f(ms[i] - ref);
        l += ls[i] * f;
        o += os[i] * f;
    }
    if constexpr (GR > 1) {
        float *mine = lds + threadIdx.x;
        mine[0] = top, mine[T] = l;
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[(2 + e) * T] = o[e];
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
            const float f = __builtin_amdgcn_exp2f(p[k * QUADS] - base);
            l += p[k * QUADS + T] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += p[k * QUADS + (2 + e) * T] * f;
        }
    }
    if (at >= all_rows || 4 * quad >= a.hd) return;
    const uint32_t g = row / R, r = row % R, tok = r / per;
    const bool any = l != 0.0f || sees_any(a, tok);
    *reinterpret_cast<u32x2 *>(a.out + ((size_t)tok * a.nh + g * per + r % per) * a.hd + 4 * quad) = finish(o, l, any);
}

template <int HD>
int launch_merge(const MxAttn &a, hipStream_t st) {
    if (a.splits < 2) return RENG_HIP_OK;
    const uint32_t rows = a.tokens * a.nh;
    constexpr uint32_t PER = 256 / (HD / 4);
    if (a.splits > MERGE_SPLITS)
        hipLaunchKernelGGL((attention_mxfp4_merge<HD, 4>), dim3(rows), dim3(HD / 4 * 4), 0, st, a);
    else
        hipLaunchKernelGGL((attention_mxfp4_merge<HD, 1>), dim3((rows + PER - 1) / PER), dim3(256), 0, st, a);
    return check_launch("attention_mxfp4_merge");
}

unsigned grid_of(const MxAttn &a) { return (a.units + MXA_XCDS - 1) / MXA_XCDS * MXA_XCDS * a.row_blocks; }

template <int HD, int NW>
int launch_rows(const MxAttn &a, hipStream_t st) {
    constexpr int LDS = NW * MXA_TILE * 2 * HD;
    static_assert(LDS <= 160 * 1024, "LDS");
    hipLaunchKernelGGL((attention_mxfp4<HD, NW>), dim3(grid_of(a)), dim3(64 * NW), LDS, st, a);
    if (int rc = check_launch("attention_mxfp4")) return rc;
    return launch_merge<HD>(a, st);
}

template <int HD, int RW, int KW, int TK, int S>
int launch_tiles(const MxAttn &a, hipStream_t st) {
    using T = MxShape<HD, RW, KW, TK, S>;
    hipLaunchKernelGGL((attention_mxfp4_tiles<HD, RW, KW, TK, S>), dim3(grid_of(a)), dim3(64 * T::W), T::LDS, st, a);
    if (int rc = check_launch("attention_mxfp4_tiles")) return rc;
    return launch_merge<HD>(a, st);
}

template <int HD>
int launch_form(const MxAttn &a, int form, hipStream_t st) {
    if constexpr (HD == 256) {
        switch (form) {
        case MXA_ROWS_16: return launch_rows<HD, 4>(a, st);
        case MXA_TILES_64: return launch_tiles<HD, 2, 2, 32, 2>(a, st);
        default: return launch_tiles<HD, 4, 1, 32, 2>(a, st);
        }
    } else {
        switch (form) {
        case MXA_ROWS_16: return launch_rows<HD, 8>(a, st);
        case MXA_TILES_64: return launch_tiles<HD, 2, 4, 32, 2>(a, st);
        case MXA_TILES_128: return launch_tiles<HD, 4, 2, 32, 2>(a, st);
        default: return launch_tiles<HD, 8, 1, 64, 4>(a, st);
        }
    }
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
    RENG_REQUIRE(fabsf(scale) <= 0x1p127f, "scale %g is above 2^127: times log2 e it leaves f32", (double)scale);
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
    if (p.hdp == 256) return launch_form<256>(a, p.form, st);
    return p.hdp == 128 ? launch_form<128>(a, p.form, st) : launch_form<64>(a, p.form, st);
}
