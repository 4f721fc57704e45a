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
#include "common.h"

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

// The general form, any even head size up to 1024 and any 4-byte alignment: a
// workgroup a token and head, 256 rows at a time, a thread a row for the scores
// and a dimension pair for the values.
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
    uint32_t *out = reinterpret_cast<uint32_t *>(a.out + ((size_t)i * a.nh + h) * a.hd);
#pragma unroll
    for (int x = 0; x < ANY_DP; ++x) {
        const uint32_t d = tid + x * ANY_T;
        if (d < pairs)
            out[d] = any ? f32_to_bf16_bits(o[x][0] / l) | (f32_to_bf16_bits(o[x][1] / l) << 16) : 0u;
    }
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API size_t reng_hip_attention_tree_workspace_bytes(size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                                            size_t len, size_t tokens) {
    (void)n_heads, (void)n_kv_heads, (void)head_dim, (void)len, (void)tokens;
    return 0;
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
    const size_t need = reng_hip_attention_tree_workspace_bytes(n_heads, n_kv_heads, head_dim, len, tokens);
    RENG_REQUIRE(workspace_bytes >= need, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    RENG_REQUIRE(need == 0 || workspace, "null workspace");
    RENG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "workspace must be 16-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const TreeArgs a{q, k_cache, v_cache, (uint32_t)n_heads, (uint32_t)n_kv_heads, (uint32_t)head_dim, (uint32_t)len,
                     (uint32_t)tokens, mask, (uint32_t)((tokens + 31) / 32), scale, out};
    hipLaunchKernelGGL(attention_tree_any, dim3((unsigned)(tokens * n_heads)), dim3(ANY_T), 0, st, a);
    return check_launch("attention_tree_any");
}
