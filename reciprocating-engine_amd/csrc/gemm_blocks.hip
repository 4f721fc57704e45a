// gemm_blocks.hip - fp8 x fp8 product with a scale for each block of 128 k:
//
//   out[m, n] = bf16(sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} dec(a[m, k]) dec(b[n, k]))
//
// a [M, K], b [N, K] codes, sa [M, KB], sb [ceil(N / 128), KB], KB = ceil(K / 128).
// The matrix cores sum a block's products; the block's sum times its scale is
// added to an f32 accumulator, so the scales cost one multiply-add per output and
// block beside 128 multiply-adds on the matrix cores.
#include "common.h"

namespace reng {
namespace {

constexpr uint32_t KBLK = 128;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct BlockArgs {
    const uint8_t *a;
    const float *sa;
    const uint8_t *b;
    const float *sb;
    uint32_t M, N, K;
    uint16_t *out;
};

__device__ __forceinline__ i32x8 join(const u32x4 &x, const u32x4 &y) {
    return i32x8{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
}

// A workgroup computes 16 MT rows of a by 16 rows of b; its waves take the
// blocks of k in turn and their sums meet in LDS. v_mfma_f32_16x16x128 with the
// weight as the first operand: lane l holds row l % 16 of either operand, and of
// the 128 codes the chunks of 16 at 16 (l / 16) and 64 + 16 (l / 16) (the same
// places for both, so the order of k within the block is free); the result's lane
// has activation row l % 16 and the four weight rows from 4 (l / 16).
template <int FA, int FB, int MT, int W>
__global__ __launch_bounds__(64 * W) void gemm_blocks_rows(BlockArgs g, uint32_t tiles_m, uint64_t tiles) {
    __shared__ f32x4 part[W][MT][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q = lane >> 4;
    const uint32_t KB = (g.K + KBLK - 1) / KBLK;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t m0 = (uint32_t)(t % tiles_m) * (16 * MT), n0 = (uint32_t)(t / tiles_m) * 16;
        // Rows past the edges are clamped and not stored.
        const uint8_t *pb = g.b + (size_t)min(n0 + row, g.N - 1) * g.K + 16 * q;
        const float *ps = g.sb + (size_t)(n0 / KBLK) * KB;
        const uint8_t *pa[MT];
        const float *psa[MT];
        f32x4 acc[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const size_t m = min(m0 + 16 * i + row, g.M - 1);
            pa[i] = g.a + m * g.K + 16 * q;
            psa[i] = g.sa + m * KB;
            acc[i] = f32x4{0, 0, 0, 0};
        }
        for (uint32_t kb = wave; kb < KB; kb += W) {
            const uint32_t k = kb * KBLK + 16 * q;
            const bool lo = k < g.K, hi = k + 64 < g.K;   // K is a multiple of 16
            const size_t ko = (size_t)kb * KBLK;
            const u32x4 z{0, 0, 0, 0};
            const i32x8 fb = join(lo ? *reinterpret_cast<const u32x4 *>(pb + ko) : z,
                                  hi ? *reinterpret_cast<const u32x4 *>(pb + ko + 64) : z);
            const float s = ps[kb];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const i32x8 fa = join(lo ? *reinterpret_cast<const u32x4 *>(pa[i] + ko) : z,
                                      hi ? *reinterpret_cast<const u32x4 *>(pa[i] + ko + 64) : z);
                const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, f32x4{0, 0, 0, 0}, FB, FA, 0,
                                                                                0, 0, 0);
                const float sc = psa[i][kb] * s;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(d[e], sc, acc[i][e]);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
        __syncthreads();
        for (uint32_t i = wave; i < MT; i += W) {
            f32x4 v = part[0][i][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) v += part[w][i][lane];
            const uint32_t m = m0 + 16 * i + row;
            if (m < g.M)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n0 + 4 * q + e < g.N)
                        g.out[(size_t)m * g.N + n0 + 4 * q + e] = (uint16_t)f32_to_bf16_bits(v[e]);
        }
        __syncthreads();   // part is written again for the next tile
    }
}

template <int FA, int FB>
int launch_blocks(const BlockArgs &g, hipStream_t st) {
    constexpr int W = 8;
    const uint64_t tiles_n = (g.N + 15) / 16;
    auto go = [&](auto mt_c) {
        constexpr int MT = decltype(mt_c)::value;
        const uint32_t tiles_m = (g.M + 16 * MT - 1) / (16 * MT);
        const uint64_t tiles = tiles_n * tiles_m, most = 1u << 20;
        hipLaunchKernelGGL((gemm_blocks_rows<FA, FB, MT, W>), dim3((unsigned)(tiles < most ? tiles : most)),
                           dim3(64 * W), 0, st, g, tiles_m, tiles);
    };
    if (g.M <= 16) go(std::integral_constant<int, 1>{});
    else if (g.M <= 32) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
    return check_launch("gemm_blocks_rows");
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API int reng_hip_gemm_fp8_blocks(const uint8_t *a, int a_format, const float *scale_a, const uint8_t *b,
                                          int b_format, const float *scale_b, size_t M, size_t N, size_t K,
                                          uint16_t *out, void *stream) {
    clear_error();
    auto valid = [](int f) { return f == RENG_HIP_E4M3 || f == RENG_HIP_E5M2; };
    RENG_REQUIRE(valid(a_format) && valid(b_format), "unknown fp8 format");
    RENG_REQUIRE(M > 0 && N > 0 && K > 0, "empty product %zu x %zu x %zu", M, N, K);
    RENG_REQUIRE(K % 16 == 0, "K = %zu is not a multiple of 16", K);
    RENG_REQUIRE(M <= 0x7fffffff && N <= 0x7fffffff && K <= 0x7fffffff, "dimension too large");
    RENG_REQUIRE(a && b && scale_a && scale_b && out, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0,
                 "a and b must be 16-byte aligned");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(scale_a) | reinterpret_cast<uintptr_t>(scale_b)) & 3) == 0 &&
                     (reinterpret_cast<uintptr_t>(out) & 1) == 0,
                 "a pointer is not aligned to its elements");
    const BlockArgs g{a, scale_a, b, scale_b, (uint32_t)M, (uint32_t)N, (uint32_t)K, out};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a_format == RENG_HIP_E4M3)
        return b_format == RENG_HIP_E4M3 ? launch_blocks<0, 0>(g, st) : launch_blocks<0, 1>(g, st);
    return b_format == RENG_HIP_E4M3 ? launch_blocks<1, 0>(g, st) : launch_blocks<1, 1>(g, st);
}
