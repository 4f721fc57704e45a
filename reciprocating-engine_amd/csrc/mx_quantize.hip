// mx_quantize.hip - MXFP4 codes and scales of a matrix (mx.h has the formula),
// and the values of such codes: of a matrix, or of a cache's rows.
//
// Bound: HBM. The quantizer reads a value once (2 or 4 bytes) and writes 17/32 of a
// byte; a lane holds 8 values, four lanes a block, sixteen the 128 columns whose four
// scales are a word. bf16 [14336, 4096]: 26.6 us (5.6 TB/s), the values back 22.6 us (6.5), f32
// 52.8 us (5.0); a copy of 1 GiB reaches 5.1. 24 rows of 18944: 2.9 and 2.6 us, the launch. Odd widths and
// rows that are not aligned go by single values: bf16 [14336, 4095] 70.6 us, back 76.4, f32 106.
#include "mx.h"

namespace reng {
namespace {

using namespace mx;

constexpr uint32_t UNIT = 128, LANES = 16;   // columns of a scale word, and the lanes that hold them

// Eight values of a row from column c on, zeros past cols.
template <typename InT, bool VEC>
__device__ __forceinline__ void load8(const InT *row, size_t c, size_t cols, float (&x)[8]) {
    if constexpr (VEC) {
        if (c < cols) {
            if constexpr (sizeof(InT) == 2) {
                const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(row + c));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] = __uint_as_float(v[i] << 16);
                    x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(row + c) + h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[4 * h + i] = __uint_as_float(v[i]);
                }
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = 0.0f;
        if constexpr (!VEC) {
            if (c + i < cols) {
                if constexpr (sizeof(InT) == 2) x[i] = __uint_as_float((uint32_t)row[c + i] << 16);
                else x[i] = row[c + i];
            }
        }
    }
}

// VEC: cols a multiple of 8, 16-byte aligned rows, 4-byte aligned codes.
template <typename InT, bool VEC>
__global__ __launch_bounds__(256) void quantize_mx(const InT *__restrict__ w, size_t rows, size_t cols, size_t ld,
                                                   size_t units, uint8_t *__restrict__ codes,
                                                   uint32_t *__restrict__ scales) {
    const size_t total = rows * units, step = (size_t)gridDim.x * (256 / LANES), pitch = (cols + 1) / 2;
    const uint32_t li = threadIdx.x % LANES;
    const size_t first = (size_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    size_t r = first / units, k = first % units;
    const size_t step_r = step / units, step_k = step % units;
    // The bound is on the workgroup's first unit, so that every lane of a wave takes part in
    // the lane exchanges.
    for (size_t g0 = (size_t)blockIdx.x * (256 / LANES); g0 < total; g0 += step) {
        const size_t u = g0 + threadIdx.x / LANES;
        const bool on = u < total;
        const size_t row = on ? r : 0, c = on ? k * UNIT + li * 8 : cols;
        float x[8];
        load8<InT, VEC>(w + row * ld, c, cols, x);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
        const uint32_t byte = scale_byte(quad_max(m)), word = scale_word(byte), d = encode8(x, byte);
        if (li == 0 && on) scales[u] = word;
        uint8_t *out = codes + row * pitch;
        if constexpr (VEC) {
            if (c < cols) *reinterpret_cast<uint32_t *>(out + c / 2) = d;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + 2 * i < cols) out[c / 2 + i] = (uint8_t)(d >> (8 * i));
        }
        r += step_r;
        k += step_k;
        if (k >= units) k -= units, ++r;
    }
}

// Eight values to out, the first n of them.
template <typename OutT, bool VEC>
__device__ __forceinline__ void store8(OutT *out, uint32_t d, uint32_t byte, size_t n) {
    const u32x4_t v = decode8(d, scale_operand(byte));
    if constexpr (VEC) {
        if constexpr (sizeof(OutT) == 2) {
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t *>(out));
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                __builtin_nontemporal_store(
                    u32x4_t{v[2 * h] << 16, v[2 * h] & 0xffff0000u, v[2 * h + 1] << 16, v[2 * h + 1] & 0xffff0000u},
                    reinterpret_cast<u32x4_t *>(out) + h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((size_t)i < n) {
                const uint32_t b = (v[i / 2] >> (16 * (i % 2))) & 0xffffu;
                if constexpr (sizeof(OutT) == 2) out[i] = (uint16_t)b;
                else out[i] = __uint_as_float(b << 16);
            }
    }
}

// VEC: cols a multiple of 8, 16-byte aligned outputs, 4-byte aligned codes.
template <typename OutT, bool VEC>
__global__ __launch_bounds__(256) void dequantize_mx(const uint8_t *__restrict__ codes,
                                                     const uint8_t *__restrict__ scales, size_t rows, size_t cols,
                                                     OutT *__restrict__ out) {
    const size_t groups = (cols + 7) / 8, total = rows * groups, step = (size_t)gridDim.x * 256;
    const size_t pitch = (cols + 1) / 2, sp = scale_pitch(cols);
    const size_t first = (size_t)blockIdx.x * 256 + threadIdx.x;
    size_t r = first / groups, k = first % groups;
    const size_t step_r = step / groups, step_k = step % groups;
    for (size_t i = first; i < total; i += step) {
        const uint8_t *p = codes + r * pitch + 4 * k;
        uint32_t d = 0;
        if constexpr (VEC) {
            d = *reinterpret_cast<const uint32_t *>(p);
        } else {
            for (size_t b = 0; b < 4 && 8 * k + 2 * b < cols; ++b) d |= (uint32_t)p[b] << (8 * b);
        }
        store8<OutT, VEC>(out + r * cols + 8 * k, d, scales[r * sp + k / 4], cols - 8 * k);
        r += step_r;
        k += step_k;
        if (k >= groups) k -= groups, ++r;
    }
}

// A row's heads follow each other in the output, a head's rows in the cache.
__global__ __launch_bounds__(256) void read_mx_cache(const reng_hip_mx_cache c, size_t first, size_t rows,
                                                     uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
    const bool values = blockIdx.y == 1 || !k;
    const uint8_t *codes = values ? c.v_codes : c.k_codes, *scales = values ? c.v_scales : c.k_scales;
    uint16_t *out = values ? v : k;
    const uint32_t hd = (uint32_t)c.head_dim, groups = hd / 8, heads = (uint32_t)c.n_kv_heads;
    const uint32_t sp = (uint32_t)scale_pitch(hd), width = heads * groups;
    const size_t total = rows * width, step = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const size_t row = i / width;
        const uint32_t at = (uint32_t)(i % width), g = at / groups, e = at % groups;
        const size_t src = (size_t)g * c.capacity + first + row;
        const uint32_t d = *reinterpret_cast<const uint32_t *>(codes + src * (hd / 2) + 4 * e);
        store8<uint16_t, true>(out + i * 8, d, scales[src * sp + e / 4], 8);
    }
}

unsigned grid_of(size_t items, size_t per, unsigned a_cu) {
    const size_t blocks = (items + per - 1) / per, most = (size_t)device_props().cus * a_cu;
    return (unsigned)(blocks < most ? blocks : most);
}

}  // namespace

int check_mx_cache(const reng_hip_mx_cache *c) {
    RENG_REQUIRE(c, "null cache");
    RENG_REQUIRE(c->n_kv_heads >= 1 && c->n_kv_heads <= 4096, "%zu key/value heads; expected 1 to 4096", c->n_kv_heads);
    RENG_REQUIRE(c->head_dim >= 32 && c->head_dim % 32 == 0 && c->head_dim <= 256,
                 "head_dim %zu is no multiple of 32 in [32, 256]", c->head_dim);
    RENG_REQUIRE(c->capacity >= 1 && c->capacity < (1u << 31), "a capacity of %zu rows; expected 1 to 2^31 - 1", c->capacity);
    RENG_REQUIRE(c->k_codes && c->k_scales && c->v_codes && c->v_scales, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15) == 0 &&
                     ((reinterpret_cast<uintptr_t>(c->k_scales) | reinterpret_cast<uintptr_t>(c->v_scales)) & 3) == 0,
                 "a cache's codes must be 16-byte aligned, its scales 4-byte");
    return RENG_HIP_OK;
}

}  // namespace reng

using namespace reng;

RENG_HIP_API int reng_hip_quantize_mxfp4(const void *w, int dtype, size_t rows, size_t cols, size_t ld, uint8_t *codes,
                                         uint8_t *scales, void *stream) {
    clear_error();
    RENG_REQUIRE(dtype == RENG_HIP_BF16 || dtype == RENG_HIP_F32, "unknown dtype %d", dtype);
    RENG_REQUIRE(rows > 0 && cols > 0, "empty shape %zu x %zu", rows, cols);
    RENG_REQUIRE(ld >= cols, "row pitch %zu is below %zu columns", ld, cols);
    RENG_REQUIRE(rows < (1u << 31) && ld < (1u << 31), "dimension too large");
    RENG_REQUIRE(w && codes && scales, "null pointer");
    const size_t es = dtype == RENG_HIP_BF16 ? 2 : 4;
    RENG_REQUIRE(reinterpret_cast<uintptr_t>(w) % es == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                 "w must be aligned to its elements, scales to 4 bytes");
    const bool vec = cols % 8 == 0 && ld * es % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(codes) % 4 == 0;
    const size_t units = (cols + UNIT - 1) / UNIT;
    const dim3 grid(grid_of(rows * units, 256 / LANES, 32));
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint32_t *sc = reinterpret_cast<uint32_t *>(scales);
    auto launch = [&](auto kern, auto *in) {
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, in, rows, cols, ld, units, codes, sc);
    };
    if (dtype == RENG_HIP_BF16) {
        const uint16_t *in = static_cast<const uint16_t *>(w);
        vec ? launch(quantize_mx<uint16_t, true>, in) : launch(quantize_mx<uint16_t, false>, in);
    } else {
        const float *in = static_cast<const float *>(w);
        vec ? launch(quantize_mx<float, true>, in) : launch(quantize_mx<float, false>, in);
    }
    return check_launch("quantize_mx");
}

RENG_HIP_API int reng_hip_dequantize_mxfp4(const uint8_t *codes, const uint8_t *scales, size_t rows, size_t cols,
                                           int out_dtype, void *out, void *stream) {
    clear_error();
    RENG_REQUIRE(out_dtype == RENG_HIP_BF16 || out_dtype == RENG_HIP_F32, "unknown dtype %d", out_dtype);
    RENG_REQUIRE(rows > 0 && cols > 0, "empty shape %zu x %zu", rows, cols);
    RENG_REQUIRE(rows < (1u << 31) && cols < (1u << 31), "dimension too large");
    RENG_REQUIRE(codes && scales && out, "null pointer");
    const size_t es = out_dtype == RENG_HIP_BF16 ? 2 : 4;
    RENG_REQUIRE(reinterpret_cast<uintptr_t>(out) % es == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                 "out must be aligned to its elements, scales to 4 bytes");
    const bool vec = cols % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0;
    const dim3 grid(grid_of(rows * ((cols + 7) / 8), 256, 32));
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto launch = [&](auto kern, auto *to) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, codes, scales, rows, cols, to); };
    if (out_dtype == RENG_HIP_BF16) {
        uint16_t *to = static_cast<uint16_t *>(out);
        vec ? launch(dequantize_mx<uint16_t, true>, to) : launch(dequantize_mx<uint16_t, false>, to);
    } else {
        float *to = static_cast<float *>(out);
        vec ? launch(dequantize_mx<float, true>, to) : launch(dequantize_mx<float, false>, to);
    }
    return check_launch("dequantize_mx");
}

RENG_HIP_API int reng_hip_cache_read_mxfp4(const reng_hip_mx_cache *cache, size_t first, size_t rows, uint16_t *k,
                                           uint16_t *v, void *stream) {
    clear_error();
    if (int rc = check_mx_cache(cache)) return rc;
    RENG_REQUIRE(rows > 0, "no rows");
    RENG_REQUIRE(first <= cache->capacity && rows <= cache->capacity - first, "rows %zu .. %zu of a cache of %zu", first,
                 first + rows, cache->capacity);
    RENG_REQUIRE(k || v, "null pointer");
    RENG_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
                 "k and v must be 16-byte aligned");
    const unsigned blocks = grid_of(rows * cache->n_kv_heads * cache->head_dim / 8, 256, 32);
    hipLaunchKernelGGL(read_mx_cache, dim3(blocks, k && v ? 2 : 1), dim3(256), 0, static_cast<hipStream_t>(stream), *cache,
                       first, rows, k, v);
    return check_launch("read_mx_cache");
}
