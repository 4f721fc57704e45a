// block_quantize.hip - fp8 codes with one f32 scale per block: 128 x 128 blocks
// of a weight, 1 x 128 groups of an activation row (block_scale.h has the
// formula). The operands of reng_hip_gemm_fp8_blocks.
//
// Bound: HBM, rows * cols * (in_bytes + 1) + 4 * blocks. Every value is read
// once and stays in registers between the absmax and the encode (bf16 [14336, 4096]
// in 128 x 128 blocks: 37.2 us, 4.7 TB/s, where a copy reaches 5.1, f32 57.0 us, 5.1 TB/s;
// 24 rows of 18944 in groups: 2.8 us, f32 3.2, a launch and one pass of loads; 4096 rows of
// 5120 in groups: 18.9 us, 3.4 TB/s, f32 27.9, 3.8).
#include <type_traits>

#include "block_scale.h"

namespace reng {
namespace {

using namespace blk;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The EPV consecutive values a lane takes of a row: 16 bytes, held as they are read.
template <typename InT>
struct Lane;
template <>
struct Lane<uint16_t> {
    static constexpr int EPV = 8, LANES = BLOCK / EPV;
    __device__ static void f(const u32x4 &v, float (&x)[EPV]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(v[i] << 16);
            x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
};
template <>
struct Lane<float> {
    static constexpr int EPV = 4, LANES = BLOCK / EPV;
    __device__ static void f(const u32x4 &v, float (&x)[EPV]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
    }
};

// Columns c .. c + EPV - 1 of a row, zeros past cols.
template <typename InT, bool VEC>
__device__ __forceinline__ u32x4 load_values(const InT *row, size_t c, size_t cols) {
    u32x4 v{0u, 0u, 0u, 0u};
    if constexpr (VEC) {
        if (c < cols) v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + c));
    } else {
#pragma unroll
        for (int i = 0; i < Lane<InT>::EPV; ++i)
            if (c + i < cols) {
                if constexpr (sizeof(InT) == 2) v[i / 2] |= (uint32_t)row[c + i] << (16 * (i % 2));
                else v[i] = __float_as_uint(row[c + i]);
            }
    }
    return v;
}

// PLAIN: the scale is a fast one and no value is NaN.
template <int F, int E, bool VEC, bool PLAIN>
__device__ __forceinline__ void store_codes(uint8_t *row, size_t c, size_t cols, const u32x4 &v, const Encoder &enc) {
    float x[E];
    Lane<typename std::conditional<E == 8, uint16_t, float>::type>::f(v, x);
    uint32_t d[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
        d[i] = PLAIN ? enc.quad_fast<F>(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3])
                     : enc.quad<F>(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    if constexpr (VEC) {
        if (c >= cols) return;
        if constexpr (E == 8) *reinterpret_cast<u32x2 *>(row + c) = u32x2{d[0], d[1]};
        else *reinterpret_cast<uint32_t *>(row + c) = d[0];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < cols) row[c + i] = (uint8_t)(d[i / 4] >> (8 * (i % 4)));
    }
}

// The largest magnitude's bits; NaN patterns sort above infinity's.
template <typename InT>
__device__ __forceinline__ uint32_t values_max(const u32x4 &v) {
    float x[Lane<InT>::EPV];
    Lane<InT>::f(v, x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < Lane<InT>::EPV; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}
// The same with NaN ignored.
template <typename InT>
__device__ __forceinline__ uint32_t values_max_no_nan(const u32x4 &v) {
    float x[Lane<InT>::EPV];
    Lane<InT>::f(v, x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < Lane<InT>::EPV; ++i) m = max(m, mag_no_nan(x[i]));
    return m;
}

// 1 x 128 groups: 16 (bf16) or 32 (f32) lanes a group, neighbouring groups in
// neighbouring lanes, grid-strided.
template <typename InT, int F, bool VEC>
__global__ __launch_bounds__(256) void quantize_groups(const InT *__restrict__ w, size_t rows, size_t cols, size_t ld,
                                                       size_t groups, float full, uint8_t *__restrict__ codes,
                                                       float *__restrict__ scales) {
    constexpr int E = Lane<InT>::EPV, L = Lane<InT>::LANES;
    const size_t total = rows * groups, step = (size_t)gridDim.x * (256 / L);
    const uint32_t gl = threadIdx.x % L;
    // Row and group in the row, carried along.
    const size_t first = (size_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    size_t r = first / groups, k = first % groups;
    const size_t step_r = step / groups, step_k = step % groups;
    // The bound is on the workgroup's first group, so that every lane of a wave takes
    // part in the lane exchange.
    for (size_t g0 = (size_t)blockIdx.x * (256 / L); g0 < total; g0 += step) {
        const size_t g = g0 + threadIdx.x / L;
        const bool on = g < total;
        const size_t row = on ? r : 0, c = on ? k * BLOCK + gl * E : cols;
        const u32x4 x = load_values<InT, VEC>(w + row * ld, c, cols);
        uint32_t m = lanes_max<L>(values_max<InT>(x));
        const bool nan = m > F32_INF;
        if (__builtin_amdgcn_ballot_w64(nan)) m = lanes_max<L>(values_max_no_nan<InT>(x));
        const float s = scale_of(m, full);
        const Encoder enc(s);
        if (__builtin_amdgcn_ballot_w64(nan || !enc.fast)) store_codes<F, E, VEC, false>(codes + row * cols, c, cols, x, enc);
        else store_codes<F, E, VEC, true>(codes + row * cols, c, cols, x, enc);
        if (on && gl == 0) scales[g] = s;
        r += step_r;
        k += step_k;
        if (k >= groups) k -= groups, ++r;
    }
}

// 128 x 128 blocks, a workgroup a block: 256 threads of 16 bytes take 16 (bf16)
// or 8 (f32) rows at a time, all 128 rows in registers.
template <typename InT, int F, bool VEC>
__global__ __launch_bounds__(256) void quantize_square(const InT *__restrict__ w, size_t rows, size_t cols, size_t ld,
                                                       uint32_t bcols, size_t blocks, float full,
                                                       uint8_t *__restrict__ codes, float *__restrict__ scales) {
    constexpr int E = Lane<InT>::EPV, L = Lane<InT>::LANES, RP = 256 / L, P = BLOCK / RP;
    __shared__ uint32_t red[4];
    for (size_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const size_t r0 = b / bcols * BLOCK + threadIdx.x / L, c = b % bcols * BLOCK + threadIdx.x % L * E;
        u32x4 x[P];
        uint32_t m = 0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const size_t r = r0 + p * RP;
            x[p] = load_values<InT, VEC>(w + (r < rows ? r : 0) * ld, r < rows ? c : cols, cols);
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t a = values_max<InT>(x[p]);
            m = m > a ? m : a;
        }
        auto block_max = [&](uint32_t v) {
            v = lanes_max<64>(v);
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
            __syncthreads();
            v = max(max(red[0], red[1]), max(red[2], red[3]));
            __syncthreads();   // red is written again
            return v;
        };
        m = block_max(m);
        const bool nan = m > F32_INF;
        if (nan) {
            m = 0;
#pragma unroll
            for (int p = 0; p < P; ++p) m = max(m, values_max_no_nan<InT>(x[p]));
            m = block_max(m);
        }
        const float s = scale_of(m, full);
        const Encoder enc(s);
        if (!nan && enc.fast) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const size_t r = r0 + p * RP;
                if (r < rows) store_codes<F, E, VEC, true>(codes + r * cols, c, cols, x[p], enc);
                __builtin_amdgcn_sched_barrier(0);   // or all of the quotients are held at once
            }
        } else {
#pragma unroll 1
            for (int p = 0; p < P; ++p) {
                const size_t r = r0 + p * RP;
                const u32x4 v = load_values<InT, VEC>(w + (r < rows ? r : 0) * ld, r < rows ? c : cols, cols);
                if (r < rows) store_codes<F, E, VEC, false>(codes + r * cols, c, cols, v, enc);
            }
        }
        if (threadIdx.x == 0) scales[b] = s;
    }
}

template <typename InT, int F, bool VEC>
int launch(const void *w, size_t rows, size_t cols, size_t ld, size_t block_rows, float full, uint8_t *codes,
           float *scales, hipStream_t st) {
    const InT *src = static_cast<const InT *>(w);
    const size_t groups = (cols + BLOCK - 1) / BLOCK, most = (size_t)device_props().cus * 64;
    if (block_rows == 1) {
        const size_t per = 256 / Lane<InT>::LANES, wgs = (rows * groups + per - 1) / per;
        hipLaunchKernelGGL((quantize_groups<InT, F, VEC>), dim3((unsigned)(wgs < most ? wgs : most)), dim3(256), 0, st,
                           src, rows, cols, ld, groups, full, codes, scales);
        return check_launch("quantize_groups");
    }
    const size_t blocks = groups * ((rows + BLOCK - 1) / BLOCK);
    hipLaunchKernelGGL((quantize_square<InT, F, VEC>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0,
                       st, src, rows, cols, ld, (uint32_t)groups, blocks, full, codes, scales);
    return check_launch("quantize_square");
}

template <typename InT>
int launch_in(const void *w, size_t rows, size_t cols, size_t ld, int format, size_t block_rows, float full,
              uint8_t *codes, float *scales, hipStream_t st) {
    // Whole 16-byte loads and whole code stores in every row.
    constexpr size_t E = Lane<InT>::EPV;
    const bool vec = cols % E == 0 && ld % E == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(codes) % E == 0;
    if (format == RENG_HIP_E4M3)
        return vec ? launch<InT, RENG_HIP_E4M3, true>(w, rows, cols, ld, block_rows, full, codes, scales, st)
                   : launch<InT, RENG_HIP_E4M3, false>(w, rows, cols, ld, block_rows, full, codes, scales, st);
    return vec ? launch<InT, RENG_HIP_E5M2, true>(w, rows, cols, ld, block_rows, full, codes, scales, st)
               : launch<InT, RENG_HIP_E5M2, false>(w, rows, cols, ld, block_rows, full, codes, scales, st);
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API int reng_hip_quantize_blocks(const void *w, int dtype, size_t rows, size_t cols, size_t ld, int format,
                                          size_t block_rows, float backoff, uint8_t *codes, float *scales,
                                          void *stream) {
    clear_error();
    RENG_REQUIRE(dtype == RENG_HIP_BF16 || dtype == RENG_HIP_F32, "unknown element type %d", dtype);
    RENG_REQUIRE(format == RENG_HIP_E4M3 || format == RENG_HIP_E5M2, "unknown fp8 format %d", format);
    RENG_REQUIRE(rows > 0 && cols > 0, "empty shape %zu x %zu", rows, cols);
    RENG_REQUIRE(rows <= 0x7fffffff && cols <= 0x7fffffff && ld <= 0x7fffffff, "dimension too large");
    RENG_REQUIRE(ld >= cols, "row pitch %zu is smaller than the row of %zu", ld, cols);
    RENG_REQUIRE(block_rows == 1 || block_rows == RENG_HIP_SCALE_BLOCK, "blocks of %zu rows; expected 1 or %d",
                 block_rows, RENG_HIP_SCALE_BLOCK);
    const float full = (format == RENG_HIP_E4M3 ? Fp8<RENG_HIP_E4M3>::MAXF : Fp8<RENG_HIP_E5M2>::MAXF) * backoff;
    RENG_REQUIRE(backoff > 0.0f && full > 0.0f && full < __builtin_inff(), "backoff %g is not positive and finite",
                 (double)backoff);
    RENG_REQUIRE(w && codes && scales, "null pointer");
    RENG_REQUIRE(reinterpret_cast<uintptr_t>(w) % (dtype == RENG_HIP_BF16 ? 2 : 4) == 0 &&
                     reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                 "w and scales must be aligned to their elements");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == RENG_HIP_BF16 ? launch_in<uint16_t>(w, rows, cols, ld, format, block_rows, full, codes, scales, st)
                                  : launch_in<float>(w, rows, cols, ld, format, block_rows, full, codes, scales, st);
}
