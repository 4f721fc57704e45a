// gemm_mxfp4.hip - product of two MXFP4 matrices (mx.h):
//
//   out[m, n] = bf16(sum_k a[m, k] b[n, k])
//
// a [M, K], b [N, K] codes with a scale byte for 32 of k. v_mfma_scale_f32_16x16x128
// takes both as they lie: lane l holds row l % 16 of either operand and the block of 32 codes
// l / 16 of 128, with that block's scale byte.
#include "common.h"
#include "mx.h"

namespace reng {
namespace {

using namespace mx;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct MxArgs {
    const uint8_t *a, *sa, *b, *sb;
    uint32_t M, N, K;
    uint16_t *out;
};

constexpr int FP4 = 4;   // the matrix instructions' number of the format

__device__ __forceinline__ f32x4 mma(const u32x4 &x, uint32_t sx, const u32x4 &y, uint32_t sy, const f32x4 &c) {
    const i32x8 xv{(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0}, yv{(int)y.x, (int)y.y, (int)y.z, (int)y.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xv, yv, c, FP4, FP4, 0, (int)sx, 0, (int)sy);
}

// 16 x 16 outputs a workgroup, its four waves taking 128 of k in turn.
__global__ __launch_bounds__(256) void gemm_mx_simple(MxArgs g, uint32_t tiles_m) {
    __shared__ f32x4 sums[4][64];
    const uint32_t lane = threadIdx.x & 63, row = lane & 15, q = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t m0 = blockIdx.x % tiles_m * 16, n0 = blockIdx.x / tiles_m * 16;
    const uint32_t blocks = g.K / BLOCK, sp = (uint32_t)scale_pitch(g.K);
    const uint32_t m = min(m0 + row, g.M - 1), n = min(n0 + row, g.N - 1);   // rows past the last are not stored
    const uint8_t *pa = g.a + (size_t)m * (g.K / 2), *pb = g.b + (size_t)n * (g.K / 2);
    f32x4 acc{0, 0, 0, 0};
    for (uint32_t k = wave * 4; k < blocks; k += 16) {
        u32x4 a{0u, 0u, 0u, 0u}, b{0u, 0u, 0u, 0u};
        uint32_t sa = ONE_BYTE, sb = ONE_BYTE;
        if (k + q < blocks) {
            a = *reinterpret_cast<const u32x4 *>(pa + (k + q) * 16);
            b = *reinterpret_cast<const u32x4 *>(pb + (k + q) * 16);
            sa = g.sa[(size_t)m * sp + k + q];
            sb = g.sb[(size_t)n * sp + k + q];
        }
        acc = mma(b, sb, a, sa, acc);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < 4; ++w) acc += sums[w][lane];
    // The lane has activation row l % 16 and four weight rows.
    if (m0 + row >= g.M) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t at = n0 + 4 * q + e;
        if (at < g.N) g.out[(size_t)(m0 + row) * g.N + at] = (uint16_t)f32_to_bf16_bits(acc[e]);
    }
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API int reng_hip_gemm_mxfp4(const uint8_t *a, const uint8_t *scale_a, const uint8_t *b, const uint8_t *scale_b,
                                     size_t M, size_t N, size_t K, uint16_t *out, void *stream) {
    clear_error();
    RENG_REQUIRE(M > 0 && N > 0 && K > 0, "empty product %zu x %zu x %zu", M, N, K);
    RENG_REQUIRE(K % mx::BLOCK == 0, "K = %zu is not a multiple of %u", K, mx::BLOCK);
    // Offsets within a tile's 256 rows are 31 bits.
    RENG_REQUIRE(M <= 0x7fffffff && N <= 0x7fffffff && K <= (1u << 22), "dimension too large");
    RENG_REQUIRE(a && b && scale_a && scale_b && out, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0,
                 "a and b must be 16-byte aligned");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(scale_a) | reinterpret_cast<uintptr_t>(scale_b)) & 3) == 0 &&
                     (reinterpret_cast<uintptr_t>(out) & 1) == 0,
                 "scales must be 4-byte aligned, out to its elements");
    const MxArgs g{a, scale_a, b, scale_b, (uint32_t)M, (uint32_t)N, (uint32_t)K, out};
    const uint32_t tiles_m = (g.M + 15) / 16, tiles_n = (g.N + 15) / 16;
    RENG_REQUIRE((uint64_t)tiles_m * tiles_n * 256 < (1ull << 32), "%u x %u outputs are too many for a launch", g.M, g.N);
    hipLaunchKernelGGL(gemm_mx_simple, dim3(tiles_m * tiles_n), dim3(256), 0, static_cast<hipStream_t>(stream), g, tiles_m);
    return check_launch("gemm_mx_simple");
}
