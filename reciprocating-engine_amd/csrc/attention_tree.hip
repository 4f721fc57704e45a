// attention_tree.hip - attention of a tree of drafted tokens over a cache.
//
// The cache holds len rows of context and then the rows of T drafted tokens.
// Token i sees every context row, and drafted row j where bit j of its mask row
// is set (its ancestors and itself); without a mask the tokens are a chain and
// token i sees drafted rows 0 .. i. Per token i and query head h, with g = h /
// (n_heads / n_kv_heads), over the rows j it sees:
//
//   s_j = scale * q[i, h] . k[j, g]        p = softmax(s)        out[i, h] = sum_j p_j v[j, g]
//
// f32 inside. A row that a token does not see takes no part, whatever it holds
// (NaN and infinities included); a token that sees nothing (len = 0 and an empty
// mask row) gives zeros; a NaN score among the rows seen makes its output NaN.
// An infinity among the values seen is an infinity of the output, however small
// its row's weight, and NaN where the weight is exactly 0 (a score of -inf) or
// infinities of both signs meet: settle() decides it by this rule where a sum has
// become NaN, so that it does not depend on how the cache is cut.
#include <float.h>

#include <type_traits>

#include "common.h"
#include "mfma_pipe.h"
#include "tree_plan.h"

namespace reng {
namespace {

struct TreeArgs {
    const uint16_t *q, *k, *v;
    uint32_t nh, nkv, hd;
    uint32_t len, tokens;
    const uint32_t *mask;   // null: a chain
    uint32_t words;         // of a mask row
    float scale;
    uint16_t *out;
};

__device__ __forceinline__ float bf16f(uint32_t b) { return __uint_as_float(b << 16); }

__device__ __forceinline__ bool sees(const TreeArgs &a, uint32_t i, uint32_t j) {
    if (j < a.len) return true;
    const uint32_t d = j - a.len;
    if (d >= a.tokens) return false;
    return a.mask ? (a.mask[(size_t)i * a.words + d / 32] >> (d % 32)) & 1 : d <= i;
}

// Where a query's sums gave a NaN though its scores are numbers, an infinite value met a weight
// or a factor of 0 (its row's own, or one that underflowed against the maximum of its tile, its
// split or the whole) or an infinity of the other sign, or a value is NaN. Then the rows are gone
// over again for such values, four bits a dimension: it sees a row with +inf (1), with -inf (2),
// with NaN or with either at a weight of 0 (4). With a finite sum of weights no score seen is NaN
// or +inf, so the query holds no infinity (each of its scores would be one, or NaN), and a row's
// score is -inf exactly where its key holds one.
__device__ __forceinline__ uint32_t special(uint32_t bf16, bool weightless) {
    const uint32_t x = bf16 & 0x7fffu;
    return x < 0x7f80u ? 0u : x > 0x7f80u || weightless ? 4u : bf16 & 0x8000u ? 2u : 1u;
}
__device__ __forceinline__ bool holds_inf(uint32_t pair) {
    return (pair & 0x7fffu) == 0x7f80u || (pair & 0x7fff0000u) == 0x7f800000u;
}
// x, a sum, where it is NaN: the infinity those bits leave.
__device__ __forceinline__ float settled(float x, uint32_t bits) {
    return !__builtin_isnan(x) ? x : bits == 1 ? INFINITY : bits == 2 ? -INFINITY : x;
}

// Whether a sum of weights is a number that outputs can be formed with.
__device__ __forceinline__ bool is_sum(float l) { return l > 0.0f && l < INFINITY; }

// The general form, any even head size up to 1024 and any 4-byte alignment: a
// workgroup a token and head, 256 rows at a time, a thread a row for the scores
// and a dimension pair for the values. It loads 4 bytes a lane and does not split the
// cache (32 heads on 8 of 128 dimensions, one token after 4096 rows: 1.35 ms, where the
// tiled form takes 18.6 us).
constexpr int ANY_T = 256, ANY_DP = 1024 / 2 / ANY_T;

__global__ __launch_bounds__(ANY_T) void attention_tree_any(TreeArgs a) {
    __shared__ float qs[1024], p[ANY_T], red[2][ANY_T / 64];
    __shared__ uint8_t seen[ANY_T];
    const uint32_t tid = threadIdx.x, i = blockIdx.x / a.nh, h = blockIdx.x % a.nh, g = h / (a.nh / a.nkv);
    const uint16_t *q = a.q + ((size_t)i * a.nh + h) * a.hd;
    const size_t pitch = (size_t)a.nkv * a.hd;
    const uint16_t *kb = a.k + (size_t)g * a.hd, *vb = a.v + (size_t)g * a.hd;
    for (uint32_t d = tid; d < a.hd; d += ANY_T) qs[d] = bf16f(q[d]);
    float m = -INFINITY, l = 0.0f;
    float o[ANY_DP][2] = {};
    const uint32_t rows = a.len + a.tokens, pairs = a.hd / 2;
    bool any = false;
    __syncthreads();
    for (uint32_t j0 = 0; j0 < rows; j0 += ANY_T) {
        const uint32_t j = j0 + tid;
        const bool on = j < rows && sees(a, i, j);
        float s = -INFINITY;
        if (on) {
            const uint32_t *kr = reinterpret_cast<const uint32_t *>(kb + (size_t)j * pitch);
            float dot = 0.0f;
            for (uint32_t d = 0; d < pairs; ++d) {
                const uint32_t w = kr[d];
                dot = fmaf(qs[2 * d], bf16f(w), dot);
                dot = fmaf(qs[2 * d + 1], __uint_as_float(w & 0xffff0000u), dot);
            }
            s = dot * a.scale;
        }
        float mx = s;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
        if ((tid & 63) == 0) red[0][tid >> 6] = mx;
        seen[tid] = on;
        any |= __syncthreads_or(on);
#pragma unroll
        for (int w = 0; w < ANY_T / 64; ++w) mx = fmaxf(mx, red[0][w]);
        // With nothing above -inf so far, exponents are taken against 0: they are 0.
        const float mn = fmaxf(m, mx), at = mn == -INFINITY ? 0.0f : mn;
        const float e = on ? expf(s - at) : 0.0f;
        p[tid] = e;
        const float ps = wave_sum_f32(e);
        if ((tid & 63) == 0) red[1][tid >> 6] = ps;
        __syncthreads();
        const float c = expf(m - at);
        l *= c;
#pragma unroll
        for (int w = 0; w < ANY_T / 64; ++w) l += red[1][w];
        m = mn;
#pragma unroll
        for (int x = 0; x < ANY_DP; ++x) {
            const uint32_t d = tid + x * ANY_T;
            if (d >= pairs) break;
            o[x][0] *= c;
            o[x][1] *= c;
            const uint32_t n = min((uint32_t)ANY_T, rows - j0);
            for (uint32_t t = 0; t < n; ++t) {
                if (!seen[t]) continue;
                const uint32_t w = reinterpret_cast<const uint32_t *>(vb + (size_t)(j0 + t) * pitch)[d];
                o[x][0] = fmaf(p[t], bf16f(w), o[x][0]);
                o[x][1] = fmaf(p[t], __uint_as_float(w & 0xffff0000u), o[x][1]);
            }
        }
        __syncthreads();   // p, seen and red are written again
    }
    // l = 0: nothing seen (zeros), or every score seen is -inf (NaN, as softmax has it).
    float y[ANY_DP][2];
    bool nan = false;
#pragma unroll
    for (int x = 0; x < ANY_DP; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            y[x][e] = o[x][e] / l;
            nan |= __builtin_isnan(y[x][e]);
        }
    if (__syncthreads_or(nan && is_sum(l))) {
        uint32_t hit[ANY_DP] = {};
        for (uint32_t j0 = 0; j0 < rows; j0 += ANY_T) {
            const uint32_t j = j0 + tid, n = min((uint32_t)ANY_T, rows - j0);
            const bool on = j < rows && sees(a, i, j);
            bool weightless = false;
            if (on) {
                const uint32_t *kr = reinterpret_cast<const uint32_t *>(kb + (size_t)j * pitch);
                for (uint32_t d = 0; d < pairs; ++d) weightless |= holds_inf(kr[d]);
            }
            seen[tid] = on + (on && weightless);
            __syncthreads();
#pragma unroll
            for (int x = 0; x < ANY_DP; ++x) {
                const uint32_t d = tid + x * ANY_T;
                if (d >= pairs) break;
                for (uint32_t t = 0; t < n; ++t) {
                    if (!seen[t]) continue;
                    const uint32_t w = reinterpret_cast<const uint32_t *>(vb + (size_t)(j0 + t) * pitch)[d];
                    hit[x] |= special(w & 0xffffu, seen[t] == 2) | (special(w >> 16, seen[t] == 2) << 4);
                }
            }
            __syncthreads();   // seen is written again
        }
#pragma unroll
        for (int x = 0; x < ANY_DP; ++x)
            if (is_sum(l)) y[x][0] = settled(y[x][0], hit[x] & 7u), y[x][1] = settled(y[x][1], hit[x] >> 4);
    }
    uint32_t *out = reinterpret_cast<uint32_t *>(a.out + ((size_t)i * a.nh + h) * a.hd);
#pragma unroll
    for (int x = 0; x < ANY_DP; ++x) {
        const uint32_t d = tid + x * ANY_T;
        if (d < pairs) out[d] = any ? f32_to_bf16_bits(y[x][0]) | (f32_to_bf16_bits(y[x][1]) << 16) : 0u;
    }
}

// ------------------------------------------------------------ tiled form
//
// The query rows of a key/value head (row r: token r / per, query head r % per of
// the per that share it) go 32 to a wave. A workgroup's RW waves of a key group
// share its tiles of TK cache rows; KW key groups take tiles in turn and merge in
// LDS; splits of the cache merge in a second kernel (tree_plan.h).
//
// Per tile a wave forms S^T = K Q^T on v_mfma_f32_32x32x16_bf16 (keys from LDS
// as the first operand, the queries in registers as the second), so a lane holds
// 16 scores of one query per 32 keys: the softmax needs one exchange, with the
// lane that holds the query's other 16, and the weights are the second operand of
// O^T = V^T P^T as they lie. The weights are rounded to bf16 for that product, each by
// 2^-8 of itself at most, no more than the rounding of the output; their sum l is of the
// unrounded ones in f32. V^T comes from LDS by transposing reads. Only tiles that reach
// past the context look at the mask.
//
// Bound: HBM for few query rows on a long cache (32 heads on 8 of 128 dimensions, one
// token after 32768 rows: 38.6 us, 3.5 TB/s; 8 tokens after 131000: 108 us, 5.0 TB/s;
// a copy reaches 5.1), the matrix cores and the exponentials for many (40 on 8, a
// chain of 1024 after 16384: 357-369 us, 960-993 TFLOP/s, where a library bf16 product of
// 8192^3 reaches 1400). A tile past the context looks at its mask, a chain's too: 1024 tokens
// after 0 take 50.6 us (212 TFLOP/s), after 1024 72.5 (445). The longest chain's steps, each
// as measured when it was taken: 1050 us, the waves' halves taking turns 620, reads four
// products ahead 589, an order written out with the masked tiles in a loop of their own 477,
// splits that fill the XCDs 351 to 373. Copies issued between the weights were slower (364 ->
// 385 us).
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct TreeTiles {
    TreeArgs a;
    uint32_t row_blocks, units, splits, tiles, base, more;   // split s: base tiles, one more for the first `more`
    float *part;                                             // null: one pass
};

// Chunk (16 bytes) slots of a tile row. Keys: 32 rows are read at one chunk, so
// chunk c of row r sits in slot c ^ r. Values: 4 rows are read over 64 bytes, so
// the 64-byte quarter is permuted by the row.
template <int P2>
__device__ __forceinline__ uint32_t key_slot(uint32_t r, uint32_t c) {
    if constexpr (P2 == 8) return c ^ ((r ^ (r >> 3)) & 7);
    else return c ^ (r & 15);
}
template <int P2>
__device__ __forceinline__ uint32_t value_slot(uint32_t r, uint32_t c) {
    if constexpr (P2 == 8) return c ^ (((r >> 1) & 1) << 2);
    else return c ^ ((r & 3) << 2);
}

__device__ __forceinline__ u32x2 read_tr(const uint8_t *p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4 *)p));
}

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
}

// The value of the lane 32 further, combined.
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Bit b: whether token i sees cache row j0 + b.
__device__ __forceinline__ uint32_t seen_bits(const TreeArgs &a, uint32_t i, uint32_t j0) {
    const int d0 = (int)j0 - (int)a.len;
    int n = (a.mask ? (int)a.tokens : (int)i + 1) - d0;   // rows j0 .. j0 + n - 1 may be seen
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

__device__ bool sees_any(const TreeArgs &a, uint32_t i) {
    if (a.len || !a.mask) return true;
    for (uint32_t d = 0; d < a.tokens; ++d)
        if ((a.mask[(size_t)i * a.words + d / 32] >> (d % 32)) & 1) return true;
    return false;
}

// o / l as two bf16 pairs; l = 0: nothing seen gives zeros, scores that are all -inf give NaN.
__device__ __forceinline__ u32x2 finish(const f32x4 &o, float l, bool any) {
    if (!any) return u32x2{0u, 0u};
    const float r = 1.0f / l;   // one rounding more than a division, far below bf16's
    return u32x2{pack_bf16(o.x * r, o.y * r), pack_bf16(o.z * r, o.w * r)};
}

__device__ __forceinline__ bool any_nan(const f32x4 &o) {
    return __builtin_isnan(o.x) || __builtin_isnan(o.y) || __builtin_isnan(o.z) || __builtin_isnan(o.w);
}

// The sums o over dimensions dim .. dim + 3 of the lane's query (token tok), settled (above). Both
// halves of a wave hold queries of the same key/value head and dimensions: the lanes of a half
// that are on share the context's rows. (32 heads on 8 of 128 dimensions, one token after 32768
// rows: one of them infinite and of a weight that underflows 0.16 ms, all of them 4.1 ms.)
__device__ __forceinline__ f32x4 settle(const TreeArgs &a, uint32_t tok, uint32_t g, uint32_t dim, f32x4 o) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t half = (lane & 32) ? 0xffffffff00000000ull : 0xffffffffull;
    const uint64_t on = __builtin_amdgcn_ballot_w64(true) & half;
    const uint32_t lanes = (uint32_t)__popcll(on), mine = (uint32_t)__popcll(on & ((1ull << lane) - 1));
    const size_t pitch = (size_t)a.nkv * a.hd;
    const uint16_t *vb = a.v + (size_t)g * a.hd + dim, *kb = a.k + (size_t)g * a.hd;
    auto load = [&](uint32_t j) { return *reinterpret_cast<const u32x2 *>(vb + j * pitch); };
    auto odd = [](const u32x2 &v) {
        return special(v.x & 0xffffu, false) | special(v.x >> 16, false) | special(v.y & 0xffffu, false) |
               special(v.y >> 16, false);
    };
    auto bits = [&](uint32_t j) {
        const u32x2 v = load(j);
        if (!odd(v)) return 0u;
        bool weightless = false;
        const u32x4 *kr = reinterpret_cast<const u32x4 *>(kb + j * pitch);
        for (uint32_t d = 0; d < a.hd / 8; ++d) {
            const u32x4 k = kr[d];
            weightless |= holds_inf(k.x) || holds_inf(k.y) || holds_inf(k.z) || holds_inf(k.w);
        }
        return special(v.x & 0xffffu, weightless) | (special(v.x >> 16, weightless) << 4) |
               (special(v.y & 0xffffu, weightless) << 8) | (special(v.y >> 16, weightless) << 12);
    };
    uint32_t found = 0;
    for (uint32_t j0 = mine; j0 < a.len; j0 += 8 * lanes) {   // the context: every token sees it
        uint32_t hit = 0;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) hit |= odd(load(min(j0 + e * lanes, a.len - 1)));
        if (!hit) continue;
#pragma unroll 1
        for (uint32_t e = 0; e < 8; ++e) found |= bits(min(j0 + e * lanes, a.len - 1));
    }
    uint32_t hit = 0;
#pragma unroll
    for (uint32_t b = 0; b < 16; ++b)
        if (__builtin_amdgcn_ballot_w64((found >> b) & 1) & half) hit |= 1u << b;
    for (uint32_t d = 0; d < a.tokens; ++d)   // the drafted rows
        if (sees(a, tok, a.len + d)) hit |= bits(a.len + d);
    return f32x4{settled(o.x, hit & 7u), settled(o.y, (hit >> 4) & 7u), settled(o.z, (hit >> 8) & 7u),
                 settled(o.w, hit >> 12)};
}

// settle for all quads of a lane. Not inlined, and given the launch's arguments where they lie:
// inlined, it costs the loops registers (a chain of 1024 without context 48.4 -> 49.7 us, so 48.6).
__device__ __attribute__((noinline)) void settle_all(const TreeTiles *args, float *sums, uint32_t quads, uint32_t tok,
                                                     uint32_t g, float l) {
    const TreeArgs a = args->a;
    for (uint32_t i = 0; i < quads; ++i) {
        const uint32_t dim = 8 * i + 4 * (threadIdx.x >> 5 & 1);
        f32x4 x{sums[4 * i], sums[4 * i + 1], sums[4 * i + 2], sums[4 * i + 3]};
        if (dim >= a.hd || !__builtin_amdgcn_ballot_w64(any_nan(x) && is_sum(l))) continue;
        x = settle(a, tok, g, dim, x);
        if (is_sum(l))
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[4 * i + e] = x[e];
    }
}

template <int HD, int RW, int KW, int TK, int S>
struct TreeShape {
    static constexpr int W = RW * KW, P2 = HD <= 64 ? 8 : HD <= 128 ? 16 : 32, ROWB = 16 * P2;
    static constexpr int RPC = 64 / P2;                       // rows per 1 KB copy
    static constexpr int TILE = TK * ROWB, STAGE = 2 * TILE;  // keys then values
    static constexpr int CPW = TK / RPC / RW, LOADS = 2 * CPW;   // copies per wave, of keys; of both
    static constexpr int LDS = KW * S * STAGE;
    static constexpr int DB = HD / 32, KB = TK / 32;
    static constexpr int AHEAD = 6;                           // products whose operands are read ahead
    static constexpr bool TURNS = RW == 8;                    // the waves' halves take turns
    static_assert(!TURNS || (KW == 1 && S == 4), "one wave of each half on a SIMD, four slots");
    static_assert(TK % (RPC * RW) == 0, "copies split evenly");
    static_assert((KW - 1) * RW * (DB * 16 + 2) * 256 <= LDS, "the key groups merge in the ring");
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <int HD, int RW, int KW, int TK, int S>
__global__ __launch_bounds__(64 * RW * KW) void attention_tree_tiles(TreeTiles t) {
    using T = TreeShape<HD, RW, KW, TK, S>;
    constexpr int P2 = T::P2, ROWB = T::ROWB, DB = T::DB, KB = T::KB, AHEAD = T::AHEAD;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ uint32_t odd[2];   // step + 1 where a step's tiles hold a value that is no finite number
    const TreeArgs &a = t.a;
    // Workgroups go to the XCDs in turn: the row blocks of one split and key/value head
    // follow each other on one XCD, whose L2 gives them the rows after the first.
    const uint32_t b = blockIdx.x / TREE_XCDS, rb = b % t.row_blocks;
    const uint32_t unit = b / t.row_blocks * TREE_XCDS + blockIdx.x % TREE_XCDS;
    if (unit >= t.units) return;
    const uint32_t g = unit % a.nkv, split = unit / a.nkv;
    const uint32_t lane = threadIdx.x & 63, h = lane >> 5, ql = lane & 31;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW, kg = wave / RW;
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, rows = a.len + a.tokens;

    // This lane's query row (clamped: rows past the last are not stored).
    const uint32_t r0 = (rb * RW + rw) * 32 + ql, r = min(r0, R - 1), tok = r / per;
    const size_t qrow = (size_t)tok * a.nh + g * per + r % per;
    // scale < 0 goes into the queries' signs, so that the largest product is the largest score.
    const float c = fabsf(a.scale) * 1.44269504088896341f;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    bf16x8 qf[HD / 16];
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
        const uint32_t d = 16 * s + 8 * h;
        u32x4 v{0u, 0u, 0u, 0u};
        if (d < a.hd) v = *reinterpret_cast<const u32x4 *>(a.q + qrow * a.hd + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] ^= flip;
        qf[s] = __builtin_bit_cast(bf16x8, v);
    }

    // The split's tiles, cut for a chain at the last row its tokens see.
    const uint32_t t0 = split * t.base + min(split, t.more);
    uint32_t t1 = t0 + t.base + (split < t.more);
    if (!a.mask) {
        const uint32_t last = min((rb * RW + RW) * 32 - 1, R - 1) / per;
        t1 = min(t1, (a.len + last) / TK + 1);
    }
    const uint32_t n = t1 > t0 ? t1 - t0 : 0, steps = (n + KW - 1) / KW;

    // A tile's copies go through a buffer resource of its rows of this head: rows behind the
    // last cache row, and the chunks behind a head smaller than HD, lie outside it and arrive
    // as zeros.
    const uint32_t pitch = a.nkv * a.hd * 2, lr = lane / P2, ls = lane % P2, lrow = lr * pitch;
    uint8_t *ring = lds + kg * (S * T::STAGE);
    auto has = [&](uint32_t step) { return step * KW + kg < n; };
    auto issue = [&](uint32_t step) __attribute__((always_inline)) {
        uint8_t *slot = ring + (step % S) * T::STAGE;
        const uint32_t j0 = (t0 + step * KW + kg) * TK, left = min((uint32_t)TK, rows - j0);
        const size_t at = ((size_t)j0 * a.nkv + g) * a.hd;
        const uint32_t bytes = (left - 1) * pitch + a.hd * 2;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *)(a.k + at), 0, bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *)(a.v + at), 0, bytes, 0x00020000);
#pragma unroll
        for (int q = 0; q < T::CPW; ++q) {
            const uint32_t tr = (rw * T::CPW + q) * T::RPC, row = tr + lr;
            const uint32_t kc = key_slot<P2>(row, ls), vc = value_slot<P2>(row, ls), off = lrow + tr * pitch;
            const uint32_t none = 0x7fffffffu;   // past every resource
            pipe::copy16_buf_asm(rk, slot + tr * ROWB, kc * 8 < a.hd ? off + 16 * kc : none);
            pipe::copy16_buf_asm(rv, slot + T::TILE + tr * ROWB, vc * 8 < a.hd ? off + 16 * vc : none);
        }
    };
    if (threadIdx.x < 2) odd[threadIdx.x] = 0;
    __syncthreads();

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;   // the running maximum of the products, this lane's share of the sum

    f32x16 s[KB];       // a tile's scores, before the scale
    u32x4 pw[2 * KB];   // its weights in bf16: the 16 rows 16 u .. of each 32 as PV takes them
    uint32_t see[KB];   // of a tile past the context, bit 8 (i / 4) + i % 4: whether score i counts

    // 16 dimensions of 32 of a tile's keys as the matrix cores take them.
    auto key_frag = [&](const uint8_t *ks, int kb, int st) __attribute__((always_inline)) {
        const uint32_t row = 32 * kb + ql;
        return *reinterpret_cast<const u32x4 *>(ks + row * ROWB + key_slot<P2>(row, 2 * st + h) * 16);
    };
    const f32x16 zero = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f,
                         0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    auto weights = [&](auto masked_c, uint32_t j0) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_c)::value;
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
            const float f = !move ? 1.0f : m == -INFINITY ? 0.0f : exp2f((m - mx) * c);
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
        const u32x2 v0 = read_tr(vs + row * ROWB + value_slot<P2>(row, ch) * 16 + in);
        const u32x2 v1 = read_tr(vs + (row + 8) * ROWB + value_slot<P2>(row + 8, ch) * 16 + in);
        return u32x4{v0.x, v0.y, v1.x, v1.y};
    };
    // The outputs that a value of the tile which is no finite number reaches become NaN (settle()
    // decides at the end): per dimension and query, such values among the rows seen are counted on
    // the matrix cores. The sums go through memory, so that this seldom path asks for no
    // registers the others would miss.
    auto specials = [&](const uint8_t *vs) __attribute__((always_inline)) {
        volatile float sums[DB * 16];
#pragma unroll
        for (int i = 0; i < DB * 16; ++i) sums[i] = o[i / 16][i % 16];
#pragma unroll 1
        for (int d = 0; d < DB; ++d) {
            f32x16 cnt = zero;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x4 v = value_frag(vs, kb, u, d);
                    u32x4 isv, isp;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t z = 0, y = 0;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t x = (v[i] >> (16 * e)) & 0x7fffu;
                            const int k = 8 * u + 2 * i + e;
                            z |= x >= 0x7f80u ? 0x3f80u << (16 * e) : 0u;
                            y |= (see[kb] >> (8 * (k / 4) + k % 4)) & 1 ? 0x3f80u << (16 * e) : 0u;
                        }
                        isv[i] = z;
                        isp[i] = y;
                    }
                    cnt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, isv),
                                                                  __builtin_bit_cast(bf16x8, isp), cnt, 0, 0, 0);
                }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (cnt[i] > 0.0f) sums[16 * d + i] = __builtin_nanf("");
        }
#pragma unroll
        for (int i = 0; i < DB * 16; ++i) o[i / 16][i % 16] = sums[i];
    };
    auto tile_row = [&](uint32_t step) { return (t0 + step * KW + kg) * TK; };
    auto keys = [&](uint32_t step) { return ring + (step % S) * T::STAGE; };
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
        for (int p = 0; p < AHEAD; ++p) f[p] = read(p);
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
    auto score = [&](uint32_t step) __attribute__((always_inline)) { run(no, yes, nullptr, keys(step)); };

    // Every LDS read of this wave is done before another may overwrite what it read.
    auto barrier = [&] {
        pipe::wait_lgkm0();
        pipe::lds_barrier();
    };
    // The first `whole` steps' tiles lie within the context; the others look at the mask, in
    // a loop of their own, whose registers the first does not pay for.
    const uint32_t in = min(n, max(a.len / TK, t0) - t0), whole = in / KW;
    // This wave's copies of a step's tile have landed (those of up to BEHIND steps after it may
    // be in flight).
    constexpr int BEHIND = T::TURNS ? 1 : S - 2;
    auto landed = [&](uint32_t step) {
        if (BEHIND > 1 && has(step + 2)) pipe::wait_vmcnt<BEHIND * T::LOADS>();
        else if (BEHIND > 0 && has(step + 1)) pipe::wait_vmcnt<T::LOADS>();
        else pipe::wait_vmcnt<0>();
    };
    static_assert(BEHIND <= 2 && BEHIND * T::LOADS < 64, "vmcnt range");
    // A weight of 0 must take nothing from a row that is not seen. So the waves look through the
    // values of a tile that may hold such rows for anything that is no finite number, each at
    // the part it copied, and where a step's tiles held some (seldom) it marks the outputs that
    // see it and is replaced by 0. `odd` is told apart by step: a wave may be one step ahead of
    // another that has not read it yet.
    auto each_copied = [&](uint32_t step, auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < T::CPW; ++q)
            f(reinterpret_cast<u32x4 *>(ring + (step % S) * T::STAGE + T::TILE + (rw * T::CPW + q) * 1024 + lane * 16));
    };
    auto look = [&](uint32_t step) __attribute__((always_inline)) {
        bool found = false;
        each_copied(step, [&](const u32x4 *p) {
            const u32x4 v = *p;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                found |= (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
        });
        if (__builtin_amdgcn_ballot_w64(found) && lane == 0) odd[step & 1] = step + 1;
    };
    auto clean = [&](uint32_t step) __attribute__((always_inline)) {
        each_copied(step, [&](u32x4 *p) {
            u32x4 v = *p;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if ((v[i] & 0x7f80u) == 0x7f80u) v[i] &= 0xffff0000u;
                if ((v[i] & 0x7f800000u) == 0x7f800000u) v[i] &= 0xffffu;
            }
            *p = v;
        });
    };
    auto masked_step = [&](uint32_t step, uint32_t next) __attribute__((always_inline)) {
        const bool on = has(step);
        const uint8_t *vs = keys(step) + T::TILE;
        landed(step);
        if (on) look(step);
        barrier();   // every wave's copies have landed, and every wave is done with the slot before
        if (has(next)) issue(next);
        if (on) {
            score(step);
            weights(yes, tile_row(step));
        }
        if (odd[step & 1] == step + 1) {
            if (on) specials(vs);
            barrier();
            if (on) clean(step);
            barrier();
        }
        if (on) run(yes, no, vs, nullptr);
    };
    if constexpr (T::TURNS) {
        // The waves' two halves, one of each on a SIMD, take turns: while one half runs its
        // matrix products (a tile's values, the next tile's scores), the other half's
        // weights use the vector unit and its copies the memory pipe. A phase ends at a
        // barrier; the second half runs one phase behind. Tile i's scores are formed in phases
        // 2 i and 2 i + 1 and its values used in phases 2 i + 2 and 2 i + 3, so with four slots
        // the first half may issue tile i + 2 in phase 2 i + 1, the second tile i + 3 in phase
        // 2 i + 2. Tile i + 1 has landed before the barrier that ends phase 2 i + 1.
        const bool second = wave >= T::W / 2;
        const uint32_t far = second ? 3 : 2;
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i)
            if (i < far && has(i)) issue(i);
        if (whole) {
            pipe::wait_vmcnt<0>();
            barrier();
            if (second) barrier();
            score(0);
            for (uint32_t i = 0; i < whole; ++i) {
                if (second) landed(i + 1);
                barrier();
                if (has(i + far)) issue(i + far);
                weights(no, 0);
                if (!second) landed(i + 1);
                barrier();
                // Behind the last tile these scores are not used.
                run(yes, yes, keys(i) + T::TILE, keys(i + 1));
            }
            if (!second) barrier();
        }
        for (uint32_t i = whole; i < steps; ++i) masked_step(i, i + far);
    } else {
#pragma unroll
        for (int i = 0; i + 1 < S; ++i)
            if (has(i)) issue(i);
        uint32_t step = 0;
        for (; step < whole; ++step) {
            landed(step);
            barrier();   // every wave's copies have landed, and every wave is done with the slot before
            if (has(step + S - 1)) issue(step + S - 1);
            score(step);
            weights(no, 0);
            run(yes, no, keys(step) + T::TILE, nullptr);
        }
        for (; step < steps; ++step) masked_step(step, step + S - 1);
    }
    l = both_sum(l);
    float mc = m == -INFINITY ? -INFINITY : m * c;

    if constexpr (KW > 1) {
        // The other key groups' (o, m, l) through LDS, lane by lane.
        __syncthreads();
        float *buf = reinterpret_cast<float *>(lds);
        constexpr int PW = tree_wave_floats(HD);
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
        float f = exp2f(mc - at);
        l *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= f;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) {
            const float *w = buf + (k * RW + rw) * PW;
            f = exp2f(w[DB * 1024 + lane] - at);
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
    if (t.part) {
        float *w = t.part + ((size_t)unit * (t.row_blocks * RW) + rb * RW + rw) * tree_wave_floats(HD);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4 *>(w + (d * 4 + i) * 256 + lane * 4) =
                    f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        w[DB * 1024 + lane] = mc;
        w[DB * 1024 + 64 + lane] = l;
        return;
    }
    float zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // unless a sum is no finite number
#pragma unroll
    for (int i = 0; i < DB * 16; ++i) zeros[i % 4] = fmaf(o[i / 16][i % 16], 0.0f, zeros[i % 4]);
    const float odd_sums = (zeros[0] + zeros[1]) + (zeros[2] + zeros[3]);
    if (__builtin_amdgcn_ballot_w64(odd_sums != 0.0f && is_sum(l))) {   // through memory, as in specials
        float sums[DB * 16];
#pragma unroll
        for (int i = 0; i < DB * 16; ++i) sums[i] = o[i / 16][i % 16];
        // A launch has its arguments, one TreeTiles, at the start of this segment.
        settle_all((const TreeTiles *)__builtin_amdgcn_kernarg_segment_ptr(), sums, DB * 4, tok, g, l);
#pragma unroll
        for (int i = 0; i < DB * 16; ++i) o[i / 16][i % 16] = sums[i];
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

// Merges the splits' (o, m, l), which lie as a wave of attention_tree_tiles held them: a wave
// here takes one quad of dimensions of each of its lanes (32 rows, two quads each). With SW = 4
// the four waves of a workgroup take a quarter of the splits each and meet in LDS: few rows over
// many splits otherwise wait for one wave's chain of loads (one token after 4096 rows, in 32
// splits, 20.5 -> 15.3 us for the call).
template <int HD, int SW>
__global__ __launch_bounds__(256) void attention_tree_merge(TreeArgs a, const float *__restrict__ part,
                                                            uint32_t splits, uint32_t waves) {
    constexpr uint32_t Q = HD / 8;   // quads a lane
    __shared__ float lds[SW > 1 ? 4 * 6 * 64 : 1];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t w = SW > 1 ? blockIdx.x : blockIdx.x * 4 + wave, quad = w % Q, tile = w / Q;
    const uint32_t per = a.nh / a.nkv, R = a.tokens * per, g = tile / waves, r = tile % waves * 32 + (lane & 31);
    const uint32_t dim = 8 * quad + 4 * (lane >> 5);
    const bool on = g < a.nkv && r < R && dim < a.hd;
    const size_t step = (size_t)a.nkv * waves * tree_wave_floats(HD);   // from a split to the next
    const float *p = part + (size_t)tile * tree_wave_floats(HD), *ml = p + HD * 32 + lane;
    float top = -INFINITY, l = 0.0f;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    if (on) {
        const uint32_t s0 = SW > 1 ? wave : 0;
#pragma unroll 8
        for (uint32_t s = s0; s < splits; s += SW) top = fmaxf(top, ml[s * step]);
        const float at = top == -INFINITY ? 0.0f : top;
#pragma unroll 8
        for (uint32_t s = s0; s < splits; s += SW) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(p + s * step + quad * 256 + lane * 4);
            const float f = exp2f(ml[s * step] - at);
            l += ml[s * step + 64] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += v[e] * f;
        }
    }
    if constexpr (SW > 1) {
        float *mine = lds + wave * 384 + lane;
        mine[0] = top;
        mine[64] = l;
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[128 + 64 * e] = o[e];
        __syncthreads();
        if (wave > 0) return;
        const float *all = lds + lane;
        top = fmaxf(fmaxf(all[0], all[384]), fmaxf(all[768], all[1152]));
        const float at = top == -INFINITY ? 0.0f : top;
        l = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = exp2f(all[384 * k] - at);
            l += all[384 * k + 64] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += all[384 * k + 128 + 64 * e] * f;
        }
    }
    const uint32_t tok = min(r, R - 1) / per;
    // (g and dim are the same in all lanes of a half, so a wave without such a head or dimension
    // has no sums.)
    if (__builtin_amdgcn_ballot_w64(on && any_nan(o) && is_sum(l))) {
        const f32x4 x = settle(a, tok, g, dim, o);
        if (is_sum(l)) o = x;
    }
    if (!on) return;
    const bool any = l != 0.0f || sees_any(a, tok);
    uint16_t *out = a.out + ((size_t)tok * a.nh + g * per + r % per) * a.hd + dim;
    *reinterpret_cast<u32x2 *>(out) = finish(o, l, any);
}

template <int HD, int RW, int KW, int TK, int S>
int launch_tiles(const TreeArgs &a, const TreePlan &p, float *part, hipStream_t st) {
    using T = TreeShape<HD, RW, KW, TK, S>;
    const uint32_t units = p.splits * a.nkv;
    const TreeTiles t{a,       p.row_blocks,        units,
                      p.splits, p.tiles,             p.tiles / p.splits,
                      p.tiles % p.splits, p.splits > 1 ? part : nullptr};
    const unsigned grid = (units + TREE_XCDS - 1) / TREE_XCDS * TREE_XCDS * p.row_blocks;
    auto kern = attention_tree_tiles<HD, RW, KW, TK, S>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * T::W), T::LDS, st, t);
    if (int rc = check_launch("attention_tree_tiles")) return rc;
    const uint32_t merge = tree_merge_waves(p, a.nkv);
    if (merge == 0) return RENG_HIP_OK;
    const uint32_t waves = p.row_blocks * RW;
    const uint32_t pieces = a.nkv * waves * (HD / 8);
    if (merge == 4)
        hipLaunchKernelGGL((attention_tree_merge<HD, 4>), dim3(pieces), dim3(256), 0, st, a, part, p.splits, waves);
    else
        hipLaunchKernelGGL((attention_tree_merge<HD, 1>), dim3((pieces + 3) / 4), dim3(256), 0, st, a, part, p.splits,
                           waves);
    return check_launch("attention_tree_merge");
}

template <int HD>
int launch_form(const TreeArgs &a, const TreePlan &p, float *part, hipStream_t st) {
    if constexpr (HD == 256) {
        if (p.form == 0) return launch_tiles<256, 1, 2, 32, 2>(a, p, part, st);
        if (p.form == 1) return launch_tiles<256, 2, 2, 32, 2>(a, p, part, st);
        return launch_tiles<256, 4, 1, 32, 3>(a, p, part, st);
    } else {
        if (p.form == 0) return launch_tiles<HD, 1, 2, 32, 4>(a, p, part, st);
        if (p.form == 1) return launch_tiles<HD, 2, 4, 32, 2>(a, p, part, st);
        if (p.form == 2) return launch_tiles<HD, 4, 2, 32, 3>(a, p, part, st);
        return launch_tiles<HD, 8, 1, 64, 4>(a, p, part, st);
    }
}

int launch_tree(const TreeArgs &a, const TreePlan &p, float *part, hipStream_t st) {
    if (p.hdp == 64) return launch_form<64>(a, p, part, st);
    if (p.hdp == 96) return launch_form<96>(a, p, part, st);
    if (p.hdp == 128) return launch_form<128>(a, p, part, st);
    return launch_form<256>(a, p, part, st);
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API size_t reng_hip_attention_tree_workspace_bytes(size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                                            size_t len, size_t tokens) {
    if (n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads || n_heads > 4096 || head_dim > 1024) return 0;
    if (tokens > RENG_HIP_TREE_MAX_TOKENS) tokens = RENG_HIP_TREE_MAX_TOKENS;
    if (len > RENG_HIP_ATTENTION_MAX_LEN) len = RENG_HIP_ATTENTION_MAX_LEN;
    return tree_workspace(n_heads, n_kv_heads, head_dim, len, tokens);
}

RENG_HIP_API int reng_hip_attention_tree(const uint16_t *q, const uint16_t *k_cache, const uint16_t *v_cache,
                                         size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t len,
                                         size_t tokens, const uint32_t *mask, float scale, void *workspace,
                                         size_t workspace_bytes, uint16_t *out, void *stream) {
    clear_error();
    RENG_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0,
                 "%zu query heads are not a multiple of %zu key/value heads", n_heads, n_kv_heads);
    RENG_REQUIRE(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 1024, "head_dim %zu is not even in [2, 1024]",
                 head_dim);
    RENG_REQUIRE(tokens >= 1 && tokens <= RENG_HIP_TREE_MAX_TOKENS, "%zu tokens; expected 1 to %d", tokens,
                 RENG_HIP_TREE_MAX_TOKENS);
    RENG_REQUIRE(len <= RENG_HIP_ATTENTION_MAX_LEN && len + tokens <= RENG_HIP_ATTENTION_MAX_LEN,
                 "%zu context rows and %zu tokens; at most %d rows", len, tokens, RENG_HIP_ATTENTION_MAX_LEN);
    RENG_REQUIRE(n_heads <= 4096, "%zu query heads; at most 4096", n_heads);
    RENG_REQUIRE(q && k_cache && v_cache && out, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
                   reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out) |
                   reinterpret_cast<uintptr_t>(mask)) & 3) == 0,
                 "q, k_cache, v_cache, mask and out must be 4-byte aligned");
    const bool aligned = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
                           reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0 &&
                         (reinterpret_cast<uintptr_t>(out) & 7) == 0;
    const TreePlan p = tree_plan(n_heads, n_kv_heads, head_dim, len, tokens, aligned, (size_t)device_props().cus);
    const size_t need = p.fast ? tree_workspace(n_heads, n_kv_heads, head_dim, len, tokens) : 0;
    RENG_REQUIRE(workspace_bytes >= need, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    RENG_REQUIRE(need == 0 || workspace, "null workspace");
    RENG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "workspace must be 16-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const TreeArgs a{q, k_cache, v_cache, (uint32_t)n_heads, (uint32_t)n_kv_heads, (uint32_t)head_dim, (uint32_t)len,
                     (uint32_t)tokens, mask, (uint32_t)((tokens + 31) / 32), scale, out};
    if (p.fast) return launch_tree(a, p, static_cast<float *>(workspace), st);
    hipLaunchKernelGGL(attention_tree_any, dim3((unsigned)(tokens * n_heads)), dim3(ANY_T), 0, st, a);
    return check_launch("attention_tree_any");
}
