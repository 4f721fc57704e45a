// gemm_mxfp4.hip - product of two MXFP4 matrices (mx.h):
//
//   out[m, n] = bf16(sum_k a[m, k] b[n, k])
//
// a [M, K], b [N, K] codes with a scale byte for 32 of k. v_mfma_scale_f32_16x16x128
// takes both as they lie: lane l holds row l % 16 of either operand and the block of 32 codes
// l / 16 of 128, with that block's scale byte. One row of a runs on its diagonal, more on rings
// or tiles (mx_forms.h).
#include <type_traits>

#include "common.h"
#include "mfma_pipe.h"
#include "mx.h"
#include "mx_forms.h"
#include "tile_order.h"

namespace reng {
namespace {

using namespace mx;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct MxArgs {
    const uint8_t *a, *sa, *b, *sb;
    uint32_t M, N, K;
    uint16_t *out;
};

constexpr int FP4 = 4;   // the matrix instructions' number of the format

// H: the byte of either lane's scales that counts.
template <int H>
__device__ __forceinline__ f32x4 mma(const u32x4 &x, uint32_t sx, const u32x4 &y, uint32_t sy, const f32x4 &c) {
    const i32x8 xv{(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0}, yv{(int)y.x, (int)y.y, (int)y.z, (int)y.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xv, yv, c, FP4, FP4, H, (int)sx, H, (int)sy);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void *p, size_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (uint32_t)bytes, 0x00020000);
}
constexpr uint32_t NOTHING = 0x7fffffffu;   // an offset past every resource: the copy leaves zeros

// A stage is 256 of k: 128 bytes of codes and two words of scales a row. In LDS a row's eight
// chunks of 16 bytes are permuted (pipe::swz) and its scales lie two stages together.
constexpr uint32_t STAGE_K = 256, ROWB = 128;
constexpr int G = 2;   // stages of a scale copy

// Of a stage's fragment of 16 rows the two steps of 128 k.
struct Frag {
    u32x4 c[2];
};
__device__ __forceinline__ Frag fragment(const uint8_t *tile, uint32_t row, uint32_t q) {
    const uint8_t *p = tile + row * ROWB;
    const uint32_t w = pipe::swz<8>(row & 31);
    return Frag{*reinterpret_cast<const u32x4 *>(p + (q ^ w) * 16), *reinterpret_cast<const u32x4 *>(p + ((4 + q) ^ w) * 16)};
}

typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 bf16x4(const f32x4 &v) {
    return __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4_t));
}

// A lane's scales of a stage: of a row's two words byte q each, in the lowest bytes. Past K,
// where the codes are zeros, a scale of 1: `blocks` is how many of 32 are left from the stage on.
__device__ __forceinline__ uint32_t scale_pair(const u32x2 &w, uint32_t q) {
    return __builtin_amdgcn_perm(w.y, w.x, q | ((4 + q) << 8) | 0x0c0c0000u);
}
__device__ __forceinline__ uint32_t within(uint32_t pair, uint32_t q, uint32_t blocks) {
    return q >= blocks ? ONE_BYTE | (ONE_BYTE << 8) : 4 + q >= blocks ? (pair & 0xffu) | (ONE_BYTE << 8) : pair;
}

// ------------------------------------------------------------ one row
//
// A wave takes NR rows of b, 2048 of k at a time: lane l has block l of 32 codes of each and of a. The
// matrix instruction pairs row i of one operand, lanes i, 16 + i, 32 + i and 48 + i, with row j of
// the other: on the diagonal i = j are the products of a block with its own, whose sum, over the
// diagonal too, is the output. The rest of the tile is not used, and costs less than decoding would
// (codes to bf16 and dot products: [14336, 4096] 8.8 us). KS waves share rows and take pieces of k in
// turn. The weight's bytes and the launch are the time: [14336, 4096] 8.4 us, [4096, 14336] 8.9,
// [27648, 5120] 17.1, [4096, 4096] 3.9 (rings 9.7, 9.2, 19.6 and 4.1), [128256, 4096] 50.6, 5.5 TB/s. One
// row of b a wave takes 8.7 us on the first, four 8.7, eight 10.0; the next piece's loads ahead are
// equal. Of a more rows than one are faster on the rings on most products (two: 9.3 us, 9.9 and
// 4.6 here, 10.1, 9.3 and 4.1 there; four 12.9 and 10.1).
template <int KS>
__global__ __launch_bounds__(256) void gemm_mx_row(MxArgs g) {
    constexpr uint32_t NR = MX_ROW_NR, ROW_K = MX_ROW_K, GROUPS = 4 / KS;   // groups of rows of a workgroup
    __shared__ float sums[4 * NR];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % KS, grp = wave / KS;
    const uint32_t n0 = (blockIdx.x * GROUPS + grp) * NR, kb = g.K / 2, sp = (uint32_t)scale_pitch(g.K);
    const uint32_t pieces = (g.K + ROW_K - 1) / ROW_K;
    const uint32_t rows = n0 < g.N ? min(NR, g.N - n0) : 0;   // rows past N arrive as zeros
    const __amdgpu_buffer_rsrc_t rb = resource(g.b + (size_t)n0 * kb, (size_t)rows * kb);
    const __amdgpu_buffer_rsrc_t rsb = resource(g.sb + (size_t)n0 * sp, (size_t)rows * sp);
    const __amdgpu_buffer_rsrc_t ra = resource(g.a, kb), rsa = resource(g.sa, sp);
    f32x4 acc[NR];
#pragma unroll
    for (uint32_t i = 0; i < NR; ++i) acc[i] = f32x4{0, 0, 0, 0};
    for (uint32_t p = part; p < pieces; p += KS) {
        const uint32_t at = p * (ROW_K / 2) + lane * 16, blk = p * (ROW_K / BLOCK) + lane;
        const bool on = at < kb;   // past K zeros
        auto codes = [&](const __amdgpu_buffer_rsrc_t &r, uint32_t row) __attribute__((always_inline)) {
            return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, on ? at + row * kb : NOTHING, 0, 0));
        };
        auto scale = [&](const __amdgpu_buffer_rsrc_t &r, uint32_t row) __attribute__((always_inline)) {
            return (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, on ? blk + row * sp : NOTHING, 0, 0);
        };
        u32x4 b[NR];
        uint32_t sb[NR];
#pragma unroll
        for (uint32_t i = 0; i < NR; ++i) b[i] = codes(rb, i), sb[i] = scale(rsb, i);
        const u32x4 a = codes(ra, 0);
        const uint32_t sa = scale(rsa, 0);
#pragma unroll
        for (uint32_t i = 0; i < NR; ++i) acc[i] = mma<0>(b[i], sb[i], a, sa, acc[i]);
    }
    // Lane l has rows 4 (l / 16) + e of column l % 16.
    const uint32_t e = lane % 16 - 4 * (lane / 16);
    float sum[NR];
#pragma unroll
    for (uint32_t i = 0; i < NR; ++i) {
        const f32x4 x = acc[i];
        sum[i] = wave_sum_dpp(e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : e == 3 ? x[3] : 0.0f);
    }
    if constexpr (KS > 1) {
        if (lane == 0)
#pragma unroll
            for (uint32_t i = 0; i < NR; ++i) sums[wave * NR + i] = sum[i];
        __syncthreads();
        // A lane an output, the waves' sums in their order.
        if (part > 0 || lane >= rows) return;
        float t = sums[wave * NR + lane];
#pragma unroll
        for (uint32_t w = 1; w < KS; ++w) t += sums[(wave + w) * NR + lane];
        g.out[n0 + lane] = (uint16_t)f32_to_bf16_bits(t);
    } else {
        if (lane > 0) return;
#pragma unroll
        for (uint32_t i = 0; i < NR; ++i)
            if (i < rows) g.out[n0 + i] = (uint16_t)f32_to_bf16_bits(sum[i]);
    }
}

int launch_row(const MxArgs &g, hipStream_t st) {
    const uint32_t groups = (g.N + MX_ROW_NR - 1) / MX_ROW_NR, ks = mx_row_waves(g.N, g.K, (uint64_t)device_props().cus);
    const uint64_t wgs = ((uint64_t)groups * ks + 3) / 4;
    RENG_REQUIRE(wgs * 256 < (1ull << 32), "%u outputs are too many for a launch", g.N);
    const auto kern = ks == 1 ? gemm_mx_row<1> : ks == 2 ? gemm_mx_row<2> : gemm_mx_row<4>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)wgs), dim3(256), 0, st, g);
    return check_launch("gemm_mx_row");
}

// ------------------------------------------------------------ few rows
//
// Where the weight's bytes are the time, or larger tiles would leave CUs idle. A workgroup
// computes 16 MT rows of a by 16 NT rows of b; its KW waves split the stages of k evenly and
// their sums meet in LDS, in the waves' order. A wave copies its own stages through a ring of
// its own, S - 1 of them in flight, and waits for nobody until the end. The copies are 8 rows x
// 128 bytes an instruction. The weight is the matrix instruction's first operand, so the
// result's lane has activation row l % 16 and the four weight rows from 4 (l / 16).
//
// What bounds it: the fetch of the weight and, beside it, of the rows of a, which every workgroup
// brings through L2 once more: [3584, 18944] with 16, 24 and 32 rows 13.4, 15.0 and 16.2 us, one row
// by itself 10.1. What the two cost each other is not settled: with the weight in the Infinity Cache, and as
// much of a to bring, 24 rows take 9.3. Not the depth of the rings: four to eight waves of two to four
// stages take 15.2 to 15.9 at 24 rows. Operands fetched straight into registers (64 bytes of a row an
// instruction) took 18 to 23.
template <int MT, int NT, int S>
struct RingShape {
    static constexpr int ROWS = 16 * (MT + NT), STAGE = ROWS * ROWB, COPIES = ROWS / 8;
    static constexpr int SC = 2 * 1024;   // a group's scales: 64 rows of either operand
    static constexpr int WAVE = S * STAGE + 2 * SC;
    static_assert(MT <= 4 && NT <= 4, "a copy of scales holds 64 rows");
    static_assert(S <= G + 2, "a group's scales, issued ahead of a stage, land before the stage that uses them");
    static_assert(MT * NT * 1024 <= WAVE && (S - 1) * COPIES + 4 < 64, "the sums fit the ring; vmcnt range");
};

template <int MT, int NT, int KW, int S>
__global__ __launch_bounds__(64 * KW) void gemm_mx_ring(MxArgs g, uint32_t tiles_m) {
    using T = RingShape<MT, NT, S>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t lane = threadIdx.x & 63, row = lane & 15, q = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m0 = blockIdx.x % tiles_m * (16 * MT), n0 = blockIdx.x / tiles_m * (16 * NT);
    const uint32_t KB = (g.K + STAGE_K - 1) / STAGE_K, blocks = g.K / BLOCK, kb = g.K / 2, sp = (uint32_t)scale_pitch(g.K);
    const uint32_t k0 = wave * KB / KW, n = (wave + 1) * KB / KW - k0;   // this wave's stages
    // Rows past M and N and codes past K lie outside and arrive as zeros.
    const uint32_t rows_a = min((uint32_t)(16 * MT), g.M - m0), rows_b = min((uint32_t)(16 * NT), g.N - n0);
    const __amdgpu_buffer_rsrc_t ra = resource(g.a + (size_t)m0 * kb, (size_t)rows_a * kb);
    const __amdgpu_buffer_rsrc_t rb = resource(g.b + (size_t)n0 * kb, (size_t)rows_b * kb);
    const __amdgpu_buffer_rsrc_t rsa = resource(g.sa + (size_t)m0 * sp, (size_t)rows_a * sp);
    const __amdgpu_buffer_rsrc_t rsb = resource(g.sb + (size_t)n0 * sp, (size_t)rows_b * sp);
    uint8_t *ring = lds + wave * T::WAVE;
    auto issue = [&](uint32_t i) __attribute__((always_inline)) {   // stage i of this wave; past the last, nothing
        uint8_t *to = ring + i % S * T::STAGE;
        const uint32_t ko = (k0 + i) * ROWB, left = i < n ? kb - ko : 0;
#pragma unroll
        for (int c = 0; c < T::COPIES; ++c) {
            const bool of_b = c >= 2 * MT;
            const uint32_t r = (of_b ? c - 2 * MT : c) * 8 + lane / 8;
            const uint32_t ch = 16 * ((lane % 8) ^ pipe::swz<8>((c * 8 + lane / 8) & 31));
            pipe::copy16_buf_asm(of_b ? rb : ra, to + c * 1024, ch < left ? r * kb + (ko + ch) : NOTHING);
        }
    };
    auto issue_scales = [&](uint32_t grp) __attribute__((always_inline)) {   // two stages'; past a row's last, others'
        uint8_t *to = ring + S * T::STAGE + (grp & 1) * T::SC;
        const uint32_t at = lane * sp + (k0 + grp * G) * 8;
        pipe::copy16_buf_asm(rsa, to, at);
        pipe::copy16_buf_asm(rsb, to + 1024, at);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    issue_scales(0);
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
    for (uint32_t i = 0; i < n; ++i) {
        // The slot of stage i + S - 1 was read by the stage before: those reads are done.
        pipe::wait_lgkm0();
        if (i % G == 0) issue_scales(i / G + 1);
        issue(i + S - 1);
        pipe::wait_vmcnt<(S - 1) * T::COPIES>();
        asm volatile("" ::: "memory");
        const uint8_t *st = ring + i % S * T::STAGE;
        const uint8_t *sc = ring + S * T::STAGE + (i / G & 1) * T::SC + i % G * 8;
        const uint32_t left = blocks - (k0 + i) * 8;
        auto scales = [&](const uint8_t *p, uint32_t r) __attribute__((always_inline)) {
            return within(scale_pair(*reinterpret_cast<const u32x2 *>(p + r * 16), q), q, left);
        };
        Frag fb[NT];
        uint32_t sb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            fb[j] = fragment(st, 16 * (MT + j) + row, q);
            sb[j] = scales(sc + 1024, 16 * j + row);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const Frag fa = fragment(st, 16 * m + row, q);
            const uint32_t sa = scales(sc, 16 * m + row);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[m][j] = mma<0>(fb[j].c[0], sb[j], fa.c[0], sa, acc[m][j]);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[m][j] = mma<1>(fb[j].c[1], sb[j], fa.c[1], sa, acc[m][j]);
        }
    }
    pipe::wait_vmcnt<0>();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<f32x4 *>(ring + (m * NT + j) * 1024 + lane * 16) = acc[m][j];
    __syncthreads();
    const bool vec = g.N % 4 == 0 && reinterpret_cast<uintptr_t>(g.out) % 8 == 0;
    for (uint32_t t = wave; t < MT * NT; t += KW) {
        f32x4 v = *reinterpret_cast<const f32x4 *>(lds + t * 1024 + lane * 16);
#pragma unroll
        for (int w = 1; w < KW; ++w) v += *reinterpret_cast<const f32x4 *>(lds + w * T::WAVE + t * 1024 + lane * 16);
        const uint32_t m = m0 + 16 * (t / NT) + row, nn = n0 + 16 * (t % NT) + 4 * q;
        if (m >= g.M || nn >= g.N) continue;
        uint16_t *out = g.out + (size_t)m * g.N + nn;
        if (vec) {
            *reinterpret_cast<u32x2 *>(out) = bf16x4(v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (nn + e < g.N) out[e] = (uint16_t)f32_to_bf16_bits(v[e]);
        }
    }
}

template <int MT, int NT, int KW, int S>
int launch_ring(const MxArgs &g, hipStream_t st) {
    constexpr int LDS = KW * RingShape<MT, NT, S>::WAVE;
    static_assert(LDS <= 160 * 1024, "LDS");
    const uint32_t tiles_m = (g.M + 16 * MT - 1) / (16 * MT), tiles_n = (g.N + 16 * NT - 1) / (16 * NT);
    RENG_REQUIRE((uint64_t)tiles_m * tiles_n * (64 * KW) < (1ull << 32), "%u x %u outputs are too many for a launch", g.M, g.N);
    hipLaunchKernelGGL((gemm_mx_ring<MT, NT, KW, S>), dim3(tiles_m * tiles_n), dim3(64 * KW), LDS, st, g, tiles_m);
    return check_launch("gemm_mx_ring");
}

// ------------------------------------------------------------ output tiles
//
// BM x BN outputs a workgroup, WGM x WGN waves of 16 TM x 16 TN. A stage's operand rows are
// copied to an S-slot LDS ring, the scales two stages at a time. A wave keeps its TN weight
// fragments of a stage and all its scales in registers and goes through the TM activation
// fragments; the next stage's first fragments and scales are read behind the barrier before
// this stage's last two rows of products. Rows past M and N and codes past K lie outside the
// tile's buffer resources and arrive as zeros.
//
// What bounds the 256 x 256 tile: the copies, at the clock that random data leaves (3.1 PFLOP/s;
// the instruction out of registers 6.5, of zeros 8.7). [4096]^3 takes 44.5 us and [1024, 27648, 5120]
// 94; without its copies 41 and 83, without three of four products 36 and 80, with zeros for
// data 38 and 86. Tried: no turns 47 and 102, four waves of 128 x 128 43 and 96 at best.
template <int TM_, int TN_, int WGM_, int WGN_, int S_>
struct MxTile {
    static constexpr int TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, S = S_, NW = WGM * WGN;
    static constexpr int BM = 16 * TM * WGM, BN = 16 * TN * WGN;
    static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int SC = 16 * (BM + BN);   // a group's scales
    static constexpr int RING = S * STAGE + 2 * SC;
    static constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW, LOADS = LA + LB;
    static constexpr int LS = (BM + BN) / 64 / NW;   // scale copies a wave, every G stages
    static constexpr int OUT = BM * (BN * 2 + 16);   // the epilogue's rows, padded by a chunk
    static constexpr int LDS = RING > OUT ? RING : OUT;
    static constexpr bool TURNS = TM == 8;   // the halves of the rows take turns
    static_assert(!TURNS || (WGM == 2 && WGN == 4 && S == 2 && LS == 1), "a wave of each half on a SIMD");
    static_assert(LA * 8 * NW == BM && LB * 8 * NW == BN && LS * 64 * NW == BM + BN && BM % 64 == 0,
                  "copies split evenly");
    static_assert(TM % 2 == 0 && (S - 1) * LOADS + LS < 64 && S >= 2 && S <= 3 && LDS <= 160 * 1024, "vmcnt range, LDS");
};

template <typename T>
__global__ __launch_bounds__(64 * T::NW) void gemm_mx_tiles(MxArgs g, uint32_t tiles_m, uint32_t tiles, uint32_t mapm) {
    constexpr int TM = T::TM, TN = T::TN, S = T::S;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, row = lane & 15, q = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / T::WGN, wn = wave % T::WGN;
    uint32_t mt, nt;
    wide_tile_of(blockIdx.x, tiles_m, tiles, mapm, mt, nt);
    const uint32_t m0 = mt * T::BM, n0 = nt * T::BN;
    const uint32_t KB = (g.K + STAGE_K - 1) / STAGE_K, blocks = g.K / BLOCK, kb = g.K / 2, sp = (uint32_t)scale_pitch(g.K);

    const uint32_t rows_a = min((uint32_t)T::BM, g.M - m0), rows_b = min((uint32_t)T::BN, g.N - n0);
    const __amdgpu_buffer_rsrc_t ra = resource(g.a + (size_t)m0 * kb, (size_t)rows_a * kb);
    const __amdgpu_buffer_rsrc_t rb = resource(g.b + (size_t)n0 * kb, (size_t)rows_b * kb);
    const __amdgpu_buffer_rsrc_t rsa = resource(g.sa + (size_t)m0 * sp, (size_t)rows_a * sp);
    const __amdgpu_buffer_rsrc_t rsb = resource(g.sb + (size_t)n0 * sp, (size_t)rows_b * sp);
    // A copy brings 8 rows: lane l the chunk of row l / 8 that lands in slot l % 8. The whole
    // offset is the lane's (a scalar one would not count in the range check).
    auto copy_rows = [&](const __amdgpu_buffer_rsrc_t &rs, uint8_t *to, uint32_t r,
                         uint32_t step) __attribute__((always_inline)) {
        step = min(step, KB - 1);   // past the last stage: that one again, into a slot that is not read
        const uint32_t ko = step * ROWB, left = kb - ko;
        const uint32_t ch = 16 * ((lane % 8) ^ pipe::swz<8>((r + lane / 8) & 31));
        pipe::copy16_buf_asm(rs, to + r * ROWB, ch < left ? lane / 8 * kb + ch + (r * kb + ko) : NOTHING);
    };
    // N copies of a, or of b, from row 8 first on.
    auto issue_a = [&](uint32_t step, uint32_t first, auto n_c) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < decltype(n_c)::value; ++c) copy_rows(ra, lds + step % S * T::STAGE, (first + c) * 8, step);
    };
    auto issue_b = [&](uint32_t step, uint32_t first, auto n_c) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < decltype(n_c)::value; ++c)
            copy_rows(rb, lds + step % S * T::STAGE + T::A_BYTES, (first + c) * 8, step);
    };
    const std::integral_constant<int, T::LA> la{};
    const std::integral_constant<int, T::LB> lb{};
    auto issue = [&](uint32_t step) __attribute__((always_inline)) {   // a wave's share of a stage
        issue_a(step, wave * T::LA, la);
        issue_b(step, wave * T::LB, lb);
    };
    // The scales of stages G grp and G grp + 1, 64 rows a copy, a's then b's. (Those behind a row's
    // last are the next row's and are not used.)
    auto issue_scales = [&](uint32_t grp) __attribute__((always_inline)) {
        uint8_t *to = lds + S * T::STAGE + (grp & 1) * T::SC;
#pragma unroll
        for (int c = 0; c < T::LS; ++c) {
            const uint32_t w = wave * T::LS + c;
            const bool of_b = w >= T::BM / 64;
            pipe::copy16_buf_asm(of_b ? rsb : rsa, to + w * 1024, ((of_b ? w - T::BM / 64 : w) * 64 + lane) * sp + grp * (8 * G));
        }
    };

    const uint32_t sw = pipe::swz<8>(row), o0 = (q ^ sw) * 16, o1 = ((4 + q) ^ sw) * 16;
    // Rows 16 i .. of a wave's operand: the permutation's second half differs by 16 rows.
    auto frag = [&](const uint8_t *base, int i) __attribute__((always_inline)) {
        const uint32_t flip = (i & 1) ? 2 * 16 : 0;   // swz<8>(r + 16) = swz<8>(r) ^ 2
        const uint8_t *p = base + (16 * i + row) * ROWB;
        return Frag{*reinterpret_cast<const u32x4 *>(p + (o0 ^ flip)), *reinterpret_cast<const u32x4 *>(p + (o1 ^ flip))};
    };
    auto a_of = [&](uint32_t step) { return lds + (step % S) * T::STAGE + wm * (16 * TM * ROWB); };
    auto b_of = [&](uint32_t step) { return lds + (step % S) * T::STAGE + T::A_BYTES + wn * (16 * TN * ROWB); };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    constexpr int R = TM % 4 == 0 ? 4 : 2;   // activation fragments held: two rows are read ahead, or the row after next
    static_assert(TM % R == 0, "the ring of fragments keeps its place from stage to stage");
    Frag fa[R], fb[TN];
    uint32_t sa[TM], sb[TN];   // this stage's scales
    u32x2 raw[TM + TN];        // and their words as read
    auto read_scales = [&](uint32_t t) __attribute__((always_inline)) {
        const uint8_t *sc = lds + S * T::STAGE + (t / G & 1) * T::SC + t % G * 8;
#pragma unroll
        for (int i = 0; i < TM; ++i) raw[i] = *reinterpret_cast<const u32x2 *>(sc + 16 * (wm * (16 * TM) + 16 * i + row));
#pragma unroll
        for (int j = 0; j < TN; ++j)
            raw[TM + j] = *reinterpret_cast<const u32x2 *>(sc + 16 * (T::BM + wn * (16 * TN) + 16 * j + row));
    };
    auto take_scales = [&](uint32_t t) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = scale_pair(raw[i], q);
#pragma unroll
        for (int j = 0; j < TN; ++j) sb[j] = scale_pair(raw[TM + j], q);
        if (t * 8 + 8 > blocks) {
            const uint32_t left = t * 8 < blocks ? blocks - t * 8 : 0;
#pragma unroll
            for (int i = 0; i < TM; ++i) sa[i] = within(sa[i], q, left);
#pragma unroll
            for (int j = 0; j < TN; ++j) sb[j] = within(sb[j], q, left);
        }
    };
    auto product = [&](int i, int j, auto h_c, const Frag &f) __attribute__((always_inline)) {
        constexpr int H = decltype(h_c)::value;
        acc[i][j] = mma<H>(fb[j].c[H], sb[j], f.c[H], sa[i], acc[i][j]);
    };
    const std::integral_constant<int, 0> lower{};
    const std::integral_constant<int, 1> upper{};

    if constexpr (T::TURNS) {
        // The two halves of the tile's rows take turns, a wave of each on a SIMD: while one half's
        // products run, the other copies its rows of a later stage and reads the first fragments
        // of its next one. A phase ends at a barrier; the second half runs one behind. The first
        // half's products of stage t are phase 2 t, its turnover 2 t + 1, the second's 2 t + 1 and
        // 2 t + 2. Both halves have stage t's weight fragments in registers by the end of phase 2 t,
        // so in phase 2 t + 1 the first half puts its rows and the weight codes of stage t + 2 into
        // the slot, in phase 2 t + 2 the second its rows; each has landed before its next
        // products' phase ends. The scales of stages 2 g and 2 g + 1 are copied in the turnovers behind
        // products 2 g - 3, a's by the first half in phase 4 g - 5, b's by the second in 4 g - 4. They
        // have landed by the end of phase 4 g - 3 and are first read in phase 4 g - 1; their buffer was
        // last read, for stage 2 g - 3, in phases 4 g - 7 and 4 g - 6.
        auto turnover = [&](uint32_t t) __attribute__((always_inline)) {
            read_scales(t);
            take_scales(t);
            fa[0] = frag(a_of(t), 0);
            fa[1] = frag(a_of(t), 1);
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j] = frag(b_of(t), j);
        };
        auto barrier = [&]() __attribute__((always_inline)) {
            pipe::wait_lgkm0();
            pipe::lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        auto products = [&](uint32_t t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if (i + 2 < TM) fa[(i + 2) % R] = frag(a_of(t), i + 2);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    product(i, j, lower, fa[i % R]);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    product(i, j, upper, fa[i % R]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // In the accumulation registers: left to itself the compiler moves the sums about and spills in
            // the loop (so it spills 15 registers ahead of it).
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
        };
        issue_scales(0);
        issue_scales(1);
        issue(0);
        issue(1);
        pipe::wait_vmcnt<0>();
        barrier();
        if (wm == 1) barrier();
        turnover(0);
        barrier();
        for (uint32_t t = 0; t < KB; ++t) {
            products(t);
            pipe::wait_vmcnt<0>();
            barrier();
            if (t % G == 1) issue_scales((t + 3) / G);
            issue_a(t + 2, wave * T::LA, la);
            if (wm == 0) issue_b(t + 2, wave * 2 * T::LB, std::integral_constant<int, 2 * T::LB>{});
            turnover(t + 1);
            barrier();
        }
        if (wm == 0) barrier();
    } else {
        issue_scales(0);
#pragma unroll
        for (int s = 0; s < S; ++s) issue(s);
        pipe::wait_vmcnt<(S - 1) * T::LOADS>();
        pipe::lds_barrier();
        fa[0] = frag(a_of(0), 0);
        fa[1] = frag(a_of(0), 1);
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = frag(b_of(0), j);
        read_scales(0);
        for (uint32_t t = 0; t < KB; ++t) {
            take_scales(t);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if (R == 4 && i + 2 < TM) fa[(i + 2) % R] = frag(a_of(t), i + 2);
                if (i == TM - 2) {
                    // Every fragment and scale of this stage is in registers, and the next stage has
                    // landed: behind the barrier its slot is read and this stage's is written. Scales
                    // go ahead of the stage's copies, so that they have landed with the stage before.
                    pipe::wait_lgkm0();
                    pipe::wait_vmcnt<(S - 2) * T::LOADS>();
                    pipe::lds_barrier();
                    if (t % G == 0) issue_scales(t / G + 1);
                    issue(t + S);
                    read_scales(t + 1);
                }
                if (R == 4 && i >= TM - 2) fa[(i + 2) % R] = frag(a_of(t + 1), i + 2 - TM);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    product(i, j, lower, fa[i % R]);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    product(i, j, upper, fa[i % R]);
                    if (i == TM - 1) fb[j] = frag(b_of(t + 1), j);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (R == 2) fa[i % R] = i + 2 < TM ? frag(a_of(t), i + 2) : frag(a_of(t + 1), i + 2 - TM);
            }
        }
    }
    pipe::wait_vmcnt<0>();   // the copies past the last stage, before LDS holds outputs

    // Epilogue through LDS: a lane holds four consecutive columns of a row; the workgroup
    // stores whole row segments.
    __syncthreads();
    constexpr uint32_t RB = T::BN * 2 + 16;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            *reinterpret_cast<u32x2 *>(lds + (wm * (16 * TM) + 16 * i + row) * RB + 2 * (wn * (16 * TN) + 16 * j + 4 * q)) =
                bf16x4(acc[i][j]);
        }
    __syncthreads();
    constexpr uint32_t CC = T::BN / 8;
    const bool vec = g.N % 8 == 0 && reinterpret_cast<uintptr_t>(g.out) % 16 == 0;
    for (uint32_t i = tid; i < T::BM * CC; i += 64 * T::NW) {
        const uint32_t r = i / CC, c = i % CC, m = m0 + r, n = n0 + 8 * c;
        if (m >= g.M || n >= g.N) continue;
        const u32x4 v = *reinterpret_cast<const u32x4 *>(lds + r * RB + 16 * c);
        uint16_t *out = g.out + (size_t)m * g.N + n;
        if (vec) {
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(out));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < g.N) out[e] = (uint16_t)(v[e / 2] >> (16 * (e % 2)));
        }
    }
}

template <typename T>
int launch_tiles(const MxArgs &g, hipStream_t st) {
    const uint32_t tiles_m = (g.M + T::BM - 1) / T::BM, tiles_n = (g.N + T::BN - 1) / T::BN, tiles = tiles_m * tiles_n;
    RENG_REQUIRE((uint64_t)tiles_m * tiles_n * (64 * T::NW) < (1ull << 32), "%u x %u outputs are too many for a launch", g.M,
                 g.N);
    hipLaunchKernelGGL((gemm_mx_tiles<T>), dim3(tiles), dim3(64 * T::NW), T::LDS, st, g, tiles_m, tiles,
                       wide_mapm(tiles_m, tiles_n, T::BM, T::BN));
    return check_launch("gemm_mx_tiles");
}

using Tile256 = MxTile<8, 4, 2, 4, 2>;
using Tile128 = MxTile<4, 4, 2, 2, 2>;
using Tile64 = MxTile<2, 4, 2, 1, 3>;
static_assert(Tile256::BM == 256 && Tile256::BN == 256 && Tile128::BM == 128 && Tile128::BN == 128 &&
                  Tile64::BM == 64 && Tile64::BN == 64,
              "MX_COST's tiles");

int launch_product(const MxArgs &g, hipStream_t st) {
    if (g.M == 1) return launch_row(g, st);
    switch (mx_pick(g.M, g.N, g.K, (uint64_t)device_props().cus)) {
    case MX_RING_1x1: return launch_ring<1, 1, 4, 4>(g, st);
    case MX_RING_1x2: return launch_ring<1, 2, 4, 3>(g, st);
    case MX_RING_2x1: return launch_ring<2, 1, 4, 3>(g, st);
    case MX_RING_2x2: return launch_ring<2, 2, 4, 2>(g, st);
    case MX_RING_4x1: return launch_ring<4, 1, 4, 2>(g, st);
    case MX_RING_4x2: return launch_ring<4, 2, 4, 2>(g, st);
    case MX_RING_4x4: return launch_ring<4, 4, 4, 2>(g, st);
    case MX_TILE_64: return launch_tiles<Tile64>(g, st);
    case MX_TILE_128: return launch_tiles<Tile128>(g, st);
    default: return launch_tiles<Tile256>(g, st);
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
    return launch_product(g, static_cast<hipStream_t>(stream));
}
