// residual_norm.hip - the steps between two branches of a layer in one pass:
// the norm after a branch, its gate, the scaled residual add and the norm
// before the next branch. Per row, in f32:
//
//   b = d                                 the branch's output, bf16
//   b = b / sqrt(mean(b^2) + eps) * gp    with a post-norm
//   b = b * gate                          with a gate, per column or per token and column
//   h = x + residual_scale * b            the residual stream (h = x without a branch)
//   n = h / sqrt(mean(h^2) + eps) * g
//
// and n goes out as bf16, or as fp8 codes with a scale for each 128 columns
// (block_scale.h), the operand reng_hip_gemm_fp8_blocks takes.
//
// Bound: HBM (x, d, gate, h and the output once each) for many rows, the chain
// of two block sums for few. A row stays in registers from its first read to
// its last write (with post-norm and gate, fp8 out: 4096 rows of 5120 63.5 us, 4.3
// TB/s, 1024 rows 22.8 us, 3.0; a row of 4096 3.9 us, bf16 out 3.3). Loading the gate and
// the weights of the norms ahead of the first sum made a row slower (3.1 -> 4.9 us).
#include "block_scale.h"

namespace reng {
namespace {

using namespace blk;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct NormArgs {
    const float *x;
    const uint16_t *d;        // null: no branch
    const float *post_gamma;  // null: no post-norm
    const uint16_t *gate;     // null: no gate
    size_t gate_ld;           // 0: one row for all
    float residual_scale;
    const float *gamma;
    uint32_t cols;
    float eps;
    float *h;                 // may be x; null: not written (only without a branch)
    void *out;
    float *scales;            // fp8 only
    float full;
    uint32_t groups;
};

enum { OUT_E4M3 = RENG_HIP_E4M3, OUT_E5M2 = RENG_HIP_E5M2, OUT_BF16 = 2 };

__device__ __forceinline__ float bf16f(uint32_t b) { return __uint_as_float(b << 16); }

// Sum over the workgroup, to every thread. red: a slot per wave, not used by another sum.
template <int NT>
__device__ __forceinline__ float block_total(float v, float *red) {
    v = wave_sum_dpp(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += red[w];
    return s;
}

__device__ __forceinline__ float inv_rms(float sum, uint32_t cols, float eps) {
    return 1.0f / sqrtf(sum / (float)cols + eps);
}

__device__ __forceinline__ float4 bf16x4(const uint16_t *p) {
    const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
    return float4{bf16f(v.x), __uint_as_float(v.x & 0xffff0000u), bf16f(v.y), __uint_as_float(v.y & 0xffff0000u)};
}

// A workgroup a row, VPT quads of columns a thread (thread t: columns 4 t, 4 (t + NT), ...),
// cols % 4 == 0, cols <= 4 NT VPT, rows and vectors aligned for 16-byte (f32) and 8-byte (bf16)
// accesses. 32 lanes hold the 128 columns of a scale group.
template <int OUT, int NT, int VPT>
__global__ __launch_bounds__(NT) void residual_norm_vec(NormArgs a) {
    __shared__ float red[2][NT / 64];
    const size_t base = (size_t)blockIdx.x * a.cols;
    float4 h[VPT];
    float ss = 0.0f;
    if (a.d) {
        float4 b[VPT];
        const uint16_t *gate = a.gate ? a.gate + (size_t)blockIdx.x * a.gate_ld : nullptr;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const uint32_t c = 4 * (threadIdx.x + i * NT);
            b[i] = c < a.cols ? bf16x4(a.d + base + c) : float4{0, 0, 0, 0};
            h[i] = c < a.cols ? *reinterpret_cast<const float4 *>(a.x + base + c) : float4{0, 0, 0, 0};
        }
        if (a.post_gamma) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) ss = sum_sq4(ss, b[i]);
            const float inv = inv_rms(block_total<NT>(ss, red[0]), a.cols, a.eps);
            ss = 0.0f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const uint32_t c = 4 * (threadIdx.x + i * NT);
                if (c >= a.cols) continue;
                const float4 g = *reinterpret_cast<const float4 *>(a.post_gamma + c);
                b[i] = float4{b[i].x * inv * g.x, b[i].y * inv * g.y, b[i].z * inv * g.z, b[i].w * inv * g.w};
            }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const uint32_t c = 4 * (threadIdx.x + i * NT);
            if (c >= a.cols) continue;
            if (gate) {
                const float4 g = bf16x4(gate + c);
                b[i] = float4{b[i].x * g.x, b[i].y * g.y, b[i].z * g.z, b[i].w * g.w};
            }
            const float rs = a.residual_scale;
            h[i] = float4{h[i].x + rs * b[i].x, h[i].y + rs * b[i].y, h[i].z + rs * b[i].z, h[i].w + rs * b[i].w};
            *reinterpret_cast<float4 *>(a.h + base + c) = h[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const uint32_t c = 4 * (threadIdx.x + i * NT);
            h[i] = c < a.cols ? *reinterpret_cast<const float4 *>(a.x + base + c) : float4{0, 0, 0, 0};
            if (a.h && c < a.cols) *reinterpret_cast<float4 *>(a.h + base + c) = h[i];
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) ss = sum_sq4(ss, h[i]);
    const float inv = inv_rms(block_total<NT>(ss, red[1]), a.cols, a.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t c = 4 * (threadIdx.x + i * NT);
        float4 n{0, 0, 0, 0};
        if (c < a.cols) {
            const float4 g = *reinterpret_cast<const float4 *>(a.gamma + c);
            n = float4{h[i].x * inv * g.x, h[i].y * inv * g.y, h[i].z * inv * g.z, h[i].w * inv * g.w};
        }
        if constexpr (OUT == OUT_BF16) {
            if (c < a.cols)
                *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + base + c) =
                    u32x2{f32_to_bf16_bits(n.x) | (f32_to_bf16_bits(n.y) << 16),
                          f32_to_bf16_bits(n.z) | (f32_to_bf16_bits(n.w) << 16)};
        } else {
            const uint32_t m = lanes_max<32>(
                max(max(mag_no_nan(n.x), mag_no_nan(n.y)), max(mag_no_nan(n.z), mag_no_nan(n.w))));
            const float s = scale_of(m, a.full);
            const Encoder enc(s);
            if (c < a.cols) {
                *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.out) + base + c) =
                    enc.quad<OUT>(n.x, n.y, n.z, n.w);
                if (c % BLOCK == 0) a.scales[(size_t)blockIdx.x * a.groups + c / BLOCK] = s;
            }
        }
    }
}

// Any width and alignment: a wave takes the 128 columns of a group, two a lane
// (128 g + lane and 64 further), and the groups wave, wave + NT / 64, ...; each
// pass reads the row again from L2.
template <int OUT>
__global__ __launch_bounds__(1024) void residual_norm_any(NormArgs a) {
    constexpr uint32_t NT = 1024, WAVES = NT / 64;
    __shared__ float red[2][WAVES];
    const size_t base = (size_t)blockIdx.x * a.cols;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint16_t *gate = a.gate ? a.gate + (size_t)blockIdx.x * a.gate_ld : nullptr;
    float post = 1.0f;
    if (a.post_gamma) {
        float ss = 0.0f;
        for (uint32_t g = wave; g < a.groups; g += WAVES)
            for (uint32_t c = g * BLOCK + lane; c < a.cols && c < (g + 1) * BLOCK; c += 64) {
                const float b = bf16f(a.d[base + c]);
                ss += b * b;
            }
        post = inv_rms(block_total<NT>(ss, red[0]), a.cols, a.eps);
    }
    float ss = 0.0f;
    for (uint32_t g = wave; g < a.groups; g += WAVES)
        for (uint32_t c = g * BLOCK + lane; c < a.cols && c < (g + 1) * BLOCK; c += 64) {
            float h = a.x[base + c];
            if (a.d) {
                float b = bf16f(a.d[base + c]);
                if (a.post_gamma) b = b * post * a.post_gamma[c];
                if (gate) b = b * bf16f(gate[c]);
                h = h + a.residual_scale * b;
            }
            if (a.h) a.h[base + c] = h;
            ss += h * h;
        }
    const float inv = inv_rms(block_total<NT>(ss, red[1]), a.cols, a.eps);
    // Each lane reads back what it wrote itself.
    const float *src = a.h ? a.h : a.x;
    for (uint32_t g = wave; g < a.groups; g += WAVES) {
        float n[2];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t c = g * BLOCK + lane + 64 * i;
            n[i] = c < a.cols ? src[base + c] * inv * a.gamma[c] : 0.0f;
            m = max(m, mag_no_nan(n[i]));
        }
        if constexpr (OUT == OUT_BF16) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t c = g * BLOCK + lane + 64 * i;
                if (c < a.cols) static_cast<uint16_t *>(a.out)[base + c] = (uint16_t)f32_to_bf16_bits(n[i]);
            }
        } else {
            const float s = scale_of(lanes_max<64>(m), a.full);
            const uint32_t q = Encoder(s).quad<OUT>(n[0], n[1], 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t c = g * BLOCK + lane + 64 * i;
                if (c < a.cols) static_cast<uint8_t *>(a.out)[base + c] = (uint8_t)(q >> (8 * i));
            }
            if (lane == 0) a.scales[(size_t)blockIdx.x * a.groups + g] = s;
        }
    }
}

template <int OUT, int NT, int VPT>
int launch_vpt(const NormArgs &a, unsigned rows, uint32_t vpt, hipStream_t st) {
    if constexpr (VPT < 8) {
        if (vpt > VPT) return launch_vpt<OUT, NT, VPT + 1>(a, rows, vpt, st);
    }
    hipLaunchKernelGGL((residual_norm_vec<OUT, NT, VPT>), dim3(rows), dim3(NT), 0, st, a);
    return check_launch("residual_norm_vec");
}

template <int OUT>
int launch_norm(const NormArgs &a, size_t rows, hipStream_t st) {
    auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
    const uintptr_t f32s = at(a.x) | at(a.post_gamma) | at(a.gamma) | at(a.h);
    const uintptr_t bf16s = at(a.d) | at(a.gate) | (OUT == OUT_BF16 ? at(a.out) : 0);
    const bool vec = a.cols % 4 == 0 && a.gate_ld % 4 == 0 && f32s % 16 == 0 && bf16s % 8 == 0 &&
                     (OUT == OUT_BF16 || at(a.out) % 4 == 0);
    const unsigned grid = (unsigned)rows;
    auto vpt = [&](uint32_t nt) { return (a.cols + 4 * nt - 1) / (4 * nt); };
    // Few rows wait for their own chain of loads and sums, which sixteen waves make shorter; many
    // fill the chip with four each (5120 columns, fp8 out into the Infinity Cache, 256 threads /
    // 1024: 24 rows 7.7 / 4.9 us, 512 rows 12.1 / 10.5, 1024 rows 19.9 / 20.4, 4096 rows 59 / 67).
    const bool few = rows <= 2 * (size_t)device_props().cus && a.cols > 1024;
    if (vec && vpt(256) <= 8 && !few) return launch_vpt<OUT, 256, 1>(a, grid, vpt(256), st);
    if (vec && vpt(1024) <= 8) return launch_vpt<OUT, 1024, 1>(a, grid, vpt(1024), st);
    hipLaunchKernelGGL((residual_norm_any<OUT>), dim3(grid), dim3(1024), 0, st, a);
    return check_launch("residual_norm_any");
}

int norm_args(const NormArgs &a, size_t rows, size_t cols, size_t gate_ld) {
    RENG_REQUIRE(rows > 0 && cols > 0, "empty shape %zu x %zu", rows, cols);
    // A workgroup of up to 1024 threads a row, and the launch holds fewer than 2^32 of them.
    RENG_REQUIRE(rows < (1u << 22) && cols <= 0x7fffffff, "dimension too large");
    RENG_REQUIRE(a.x && a.gamma && a.out, "null pointer");
    RENG_REQUIRE(a.d || (!a.post_gamma && !a.gate), "a post-norm or a gate without a branch");
    RENG_REQUIRE(!a.d || a.h, "a branch without h to write the residual stream to");
    RENG_REQUIRE(gate_ld == 0 || (a.gate && gate_ld >= cols), "gate pitch %zu; expected 0 or at least %zu", gate_ld,
                 cols);
    RENG_REQUIRE(a.eps >= 0.0f, "eps %g is negative", (double)a.eps);
    const uintptr_t f32s = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.post_gamma) |
                           reinterpret_cast<uintptr_t>(a.gamma) | reinterpret_cast<uintptr_t>(a.h) |
                           reinterpret_cast<uintptr_t>(a.scales);
    const uintptr_t bf16s = reinterpret_cast<uintptr_t>(a.d) | reinterpret_cast<uintptr_t>(a.gate);
    RENG_REQUIRE(f32s % 4 == 0 && bf16s % 2 == 0, "a pointer is not aligned to its elements");
    return RENG_HIP_OK;
}

}  // namespace
}  // namespace reng

using namespace reng;

RENG_HIP_API int reng_hip_residual_norm_bf16(const float *x, const uint16_t *d, const float *post_gamma,
                                             const uint16_t *gate, size_t gate_ld, float residual_scale,
                                             const float *gamma, size_t rows, size_t cols, float eps, float *h,
                                             uint16_t *out, void *stream) {
    clear_error();
    const NormArgs a{x,   d, post_gamma, gate,    gate_ld, residual_scale, gamma, (uint32_t)cols,
                     eps, h, out,        nullptr, 0.0f,    (uint32_t)((cols + BLOCK - 1) / BLOCK)};
    if (int rc = norm_args(a, rows, cols, gate_ld)) return rc;
    RENG_REQUIRE(reinterpret_cast<uintptr_t>(out) % 2 == 0, "a pointer is not aligned to its elements");
    return launch_norm<OUT_BF16>(a, rows, static_cast<hipStream_t>(stream));
}

RENG_HIP_API int reng_hip_residual_norm_fp8(const float *x, const uint16_t *d, const float *post_gamma,
                                            const uint16_t *gate, size_t gate_ld, float residual_scale,
                                            const float *gamma, size_t rows, size_t cols, float eps, int format,
                                            float backoff, float *h, uint8_t *codes, float *scales, void *stream) {
    clear_error();
    RENG_REQUIRE(format == RENG_HIP_E4M3 || format == RENG_HIP_E5M2, "unknown fp8 format %d", format);
    const float full = (format == RENG_HIP_E4M3 ? Fp8<RENG_HIP_E4M3>::MAXF : Fp8<RENG_HIP_E5M2>::MAXF) * backoff;
    RENG_REQUIRE(backoff > 0.0f && full > 0.0f && full < __builtin_inff(), "backoff %g is not positive and finite",
                 (double)backoff);
    RENG_REQUIRE(scales, "null pointer");
    const NormArgs a{x,   d, post_gamma, gate,   gate_ld, residual_scale, gamma, (uint32_t)cols,
                     eps, h, codes,      scales, full,    (uint32_t)((cols + BLOCK - 1) / BLOCK)};
    if (int rc = norm_args(a, rows, cols, gate_ld)) return rc;
    return format == RENG_HIP_E4M3 ? launch_norm<OUT_E4M3>(a, rows, static_cast<hipStream_t>(stream))
                                   : launch_norm<OUT_E5M2>(a, rows, static_cast<hipStream_t>(stream));
}
