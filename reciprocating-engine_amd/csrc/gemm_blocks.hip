// gemm_blocks.hip - fp8 x fp8 product with a scale for each block of 128 k:
//
//   out[m, n] = bf16(sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} dec(a[m, k]) dec(b[n, k]))
//
// a [M, K], b [N, K] codes, sa [M, KB], sb [ceil(N / 128), KB], KB = ceil(K / 128).
// The matrix cores sum a block's products; the block's sum times its scale is
// added to an f32 accumulator, so the scales cost one multiply-add per output and
// block beside 128 multiply-adds on the matrix cores.
//
// Bound: HBM for a row ([4096, 14336]: 12.9 us, 4.5 TB/s). Some ten to 128 rows stay below
// its rate (24 rows [3584, 18944]: 20-23 us from HBM, 14.1 out of the Infinity Cache;
// 128: 38.4), though not for want of copies in flight: rings of 3, 4 and 5 slots take 20.5,
// 20.5 and 20.8 us. Then the matrix cores ([4096, 4096, 4096]: 66-69 us, 2.0 PFLOP/s;
// M = 1024 [27648, 5120]: 148-156 us, 1.9, its 432 tiles two rounds where 1.69 would do). A
// library fp8 product with one scale a tensor takes 121-125 us there, and reaches 2.63-2.68
// PFLOP/s at 8192^3.
#include <type_traits>

#include "block_forms.h"
#include "common.h"
#include "mfma_pipe.h"
#include "tile_order.h"

namespace reng {
namespace {

constexpr uint32_t KBLK = 128;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// ------------------------------------------------------------ few rows
//
// Where the weight's bytes are the time, or larger tiles would leave CUs idle: up to 16
// rows always, more where block_pick's model has it faster (128 x [3584, 18944] and 256 x
// [4096, 4096] too). A workgroup computes 16 MT rows of a, 64 at most, by 16 NT rows of b;
// its KW waves split the blocks of k evenly and their sums meet in LDS, in the waves' order.
// A wave copies its own stages (one scale block of its rows) through a ring of its own,
// S - 1 of them in flight, and waits for nobody until the end. The copies are 8 rows x 128
// bytes an instruction: read straight into registers in the matrix operand's layout the
// codes come in 64-byte pieces. Scales are copied four stages at a time.
// v_mfma_f32_16x16x128 with the weight as the first operand: lane l holds row l % 16 of
// either operand and the chunks 2 (l / 16) and 2 (l / 16) + 1 of its 128 codes; the
// result's lane has activation row l % 16 and the four weight rows from 4 (l / 16).
template <int MT, int NT, int S>
struct RingShape {
    static constexpr int ROWS = 16 * (MT + NT), STAGE = ROWS * 128, COPIES = ROWS / 8, G = 4;
    static constexpr int SC = 2 * 1024;   // a group's scales: 64 activation rows', then the weight block's
    static constexpr int WAVE = S * STAGE + 2 * SC;
    static_assert(MT * NT * 1024 <= WAVE && (S - 1) * COPIES + 2 < 64 && 16 * NT <= 128, "the sums fit the ring; vmcnt range");
};

template <int FA, int FB, int MT, int NT, int KW, int S>
__global__ __launch_bounds__(64 * KW) void gemm_blocks_ring(BlockArgs g, uint32_t tiles_m) {
    using T = RingShape<MT, NT, S>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t lane = threadIdx.x & 63, row = lane & 15, q = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m0 = blockIdx.x % tiles_m * (16 * MT), n0 = blockIdx.x / tiles_m * (16 * NT);
    const uint32_t KB = (g.K + KBLK - 1) / KBLK;
    const uint32_t k0 = wave * KB / KW, n = (wave + 1) * KB / KW - k0;   // this wave's blocks
    auto rsrc = [](const void *p, size_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (uint32_t)bytes, 0x00020000);
    };
    // Rows past M and N and codes past K lie outside and arrive as zeros.
    const uint32_t rows_a = min((uint32_t)(16 * MT), g.M - m0), rows_b = min((uint32_t)(16 * NT), g.N - n0);
    const __amdgpu_buffer_rsrc_t ra = rsrc(g.a + (size_t)m0 * g.K, (size_t)rows_a * g.K);
    const __amdgpu_buffer_rsrc_t rb = rsrc(g.b + (size_t)n0 * g.K, (size_t)rows_b * g.K);
    const __amdgpu_buffer_rsrc_t rsa = rsrc(g.sa + (size_t)m0 * KB, (size_t)rows_a * KB * 4);
    const __amdgpu_buffer_rsrc_t rsb = rsrc(g.sb + (size_t)(n0 / KBLK) * KB, (size_t)KB * 4);
    const uint32_t none = 0x7fffffffu;
    uint8_t *ring = lds + wave * T::WAVE;
    auto issue = [&](uint32_t i) __attribute__((always_inline)) {   // stage i of this wave; past the last, nothing
        uint8_t *to = ring + i % S * T::STAGE;
        const uint32_t ko = (k0 + i) * KBLK, left = i < n ? g.K - ko : 0;
#pragma unroll
        for (int c = 0; c < T::COPIES; ++c) {
            const bool of_b = c >= 2 * MT;
            const uint32_t r = (of_b ? c - 2 * MT : c) * 8 + lane / 8;
            const uint32_t ch = 16 * ((lane % 8) ^ pipe::swz<8>((c * 8 + lane / 8) & 31));
            pipe::copy16_buf_asm(of_b ? rb : ra, to + c * 1024, ch < left ? r * g.K + (ko + ch) : none);
        }
    };
    auto issue_scales = [&](uint32_t grp) __attribute__((always_inline)) {
        uint8_t *to = ring + S * T::STAGE + (grp & 1) * T::SC;
        const uint32_t k = (k0 + grp * T::G) * 4;
        pipe::copy16_buf_asm(rsa, to, lane * KB * 4 + k);
        pipe::copy16_buf_asm(rsb, to + 1024, lane == 0 ? k : none);
    };
    auto frag = [&](const uint8_t *p, int tile) __attribute__((always_inline)) {
        const uint32_t r = 16 * tile + row, w = pipe::swz<8>(r & 31);
        p += r * 128;
        return join(*reinterpret_cast<const u32x4 *>(p + (2 * q ^ w) * 16),
                    *reinterpret_cast<const u32x4 *>(p + ((2 * q + 1) ^ w) * 16));
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
        issue(i + S - 1);
        if (i % T::G == 0) issue_scales(i / T::G + 1);
        pipe::wait_vmcnt<(S - 1) * T::COPIES>();
        asm volatile("" ::: "memory");
        const uint8_t *st = ring + i % S * T::STAGE;
        const uint8_t *sc = ring + S * T::STAGE + (i / T::G & 1) * T::SC + i % T::G * 4;
        const float sb = *reinterpret_cast<const float *>(sc + 1024);
        i32x8 fb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[j] = frag(st, MT + j);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const i32x8 fa = frag(st, m);
            const float s = *reinterpret_cast<const float *>(sc + 16 * (16 * m + row)) * sb;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, f32x4{0, 0, 0, 0}, FB, FA, 0,
                                                                                0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][j][e] = fmaf(d[e], s, acc[m][j][e]);
            }
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
            *reinterpret_cast<u32x2 *>(out) = u32x2{f32_to_bf16_bits(v.x) | (f32_to_bf16_bits(v.y) << 16),
                                                    f32_to_bf16_bits(v.z) | (f32_to_bf16_bits(v.w) << 16)};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (nn + e < g.N) out[e] = (uint16_t)f32_to_bf16_bits(v[e]);
        }
    }
}

template <int FA, int FB, int MT, int NT, int KW, int S>
int launch_ring(const BlockArgs &g, hipStream_t st) {
    constexpr int LDS = KW * RingShape<MT, NT, S>::WAVE;
    static_assert(LDS <= 160 * 1024, "LDS");
    const uint32_t tiles_m = (g.M + 16 * MT - 1) / (16 * MT), tiles_n = (g.N + 16 * NT - 1) / (16 * NT);
    RENG_REQUIRE((uint64_t)tiles_m * tiles_n * (64 * KW) < (1ull << 32), "%u x %u outputs are too many for a launch", g.M, g.N);
    hipLaunchKernelGGL((gemm_blocks_ring<FA, FB, MT, NT, KW, S>), dim3(tiles_m * tiles_n), dim3(64 * KW), LDS, st, g,
                       tiles_m);
    return check_launch("gemm_blocks_ring");
}

// ------------------------------------------------------------ output tiles
//
// BM x BN outputs a workgroup, WGM x WGN waves of 16 TM x 16 TN, K in stages of one
// scale block. A stage's operand rows are copied to an
// S-slot LDS ring (16-byte chunks of a row permuted by swz, so that fragment reads
// are free of bank conflicts; the scales four stages at a time, 16 bytes of a row:
// one stage's are 4 bytes of BM different lines, which cost the copies of the codes
// 10-40%). A wave keeps its TN weight fragments of a stage in
// registers and goes through the TM activation fragments; the 16 x 16 product of a
// stage (one v_mfma_f32_16x16x128) is scaled and added to the accumulator PART
// products later, so that the vector unit works while the matrix cores do. The next
// stage's first fragments are read behind the barrier before this stage's last two
// rows of products. Rows past M and N and codes past K lie outside the tile's buffer
// resources and arrive as zeros.
template <int TM_, int TN_, int WGM_, int WGN_, int S_>
struct BlockTile {
    static constexpr int TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, S = S_, NW = WGM * WGN;
    static constexpr int BM = 16 * TM * WGM, BN = 16 * TN * WGN;
    static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int G = 4, SC = 4 * G * (BM + 64);   // scales of G stages: BM rows', then the weight's blocks'
    static constexpr int RING = S * STAGE + 2 * SC;
    static constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW, LOADS = LA + LB;
    static constexpr int LS = (BM / 64 + 1 + NW - 1) / NW;   // scale copies a wave, every G stages
    static constexpr int OUT = BM * (BN * 2 + 16);   // the epilogue's rows, padded by a chunk
    static constexpr int LDS = RING > OUT ? RING : OUT;
    static constexpr int PART = 3;
    static constexpr bool TURNS = TM == 8;   // the halves of the rows take turns
    static_assert(!TURNS || (WGM == 2 && WGN == 4 && S == 2), "a wave of each half on a SIMD");
    static_assert(LA * 8 * NW == BM && LB * 8 * NW == BN, "copies split evenly");
    static_assert(TM % 2 == 0 && 16 * TN <= 128 && 128 % (16 * TN) == 0, "a wave's columns share a scale");
    static_assert((S - 1) * LOADS < 64 && S >= 2 && S <= 3 && LDS <= 160 * 1024, "vmcnt range, LDS");
};

template <int FA, int FB, typename T>
__global__ __launch_bounds__(64 * T::NW) void gemm_blocks_tiles(BlockArgs g, uint32_t tiles_m, uint32_t tiles,
                                                                uint32_t mapm) {
    constexpr int TM = T::TM, TN = T::TN, S = T::S, PART = T::PART;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, row = lane & 15, q = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / T::WGN, wn = wave % T::WGN;
    uint32_t mt, nt;
    wide_tile_of(blockIdx.x, tiles_m, tiles, mapm, mt, nt);
    const uint32_t m0 = mt * T::BM, n0 = nt * T::BN;
    const uint32_t KB = (g.K + KBLK - 1) / KBLK, NB = (g.N + KBLK - 1) / KBLK;

    auto rsrc = [](const void *p, size_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (uint32_t)bytes, 0x00020000);
    };
    const uint32_t rows_a = min((uint32_t)T::BM, g.M - m0), rows_b = min((uint32_t)T::BN, g.N - n0);
    const uint32_t nb0 = n0 / KBLK, nbs = min((uint32_t)((T::BN + KBLK - 1) / KBLK), NB - nb0);
    const __amdgpu_buffer_rsrc_t ra = rsrc(g.a + (size_t)m0 * g.K, (size_t)rows_a * g.K);
    const __amdgpu_buffer_rsrc_t rb = rsrc(g.b + (size_t)n0 * g.K, (size_t)rows_b * g.K);
    const __amdgpu_buffer_rsrc_t rsa = rsrc(g.sa + (size_t)m0 * KB, (size_t)rows_a * KB * 4);
    const __amdgpu_buffer_rsrc_t rsb = rsrc(g.sb + (size_t)nb0 * KB, (size_t)nbs * KB * 4);
    // A copy brings 8 rows: lane l the chunk of row l / 8 that lands in slot l % 8. The whole
    // offset is the lane's (a scalar one would not count in the range check).
    auto copy_rows = [&](const __amdgpu_buffer_rsrc_t &rs, uint8_t *to, uint32_t r, uint32_t step) __attribute__((always_inline)) {
        step = min(step, KB - 1);   // past the last stage: that one again, into a slot that is not read
        const uint32_t ko = step * KBLK, left = g.K - ko;   // codes of k left
        const uint32_t ch = 16 * ((lane % 8) ^ pipe::swz<8>((r + lane / 8) & 31));
        pipe::copy16_buf_asm(rs, to + r * 128, ch < left ? lane / 8 * g.K + ch + (r * g.K + ko) : 0x7fffffffu);
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
    // The scales of stages G grp .. G grp + 3: 64 rows of a a copy, then the blocks of b.
    // (Those behind a row's last are the next row's and are not used.)
    auto issue_scales = [&](uint32_t grp) __attribute__((always_inline)) {
        uint8_t *to = lds + S * T::STAGE + (grp & 1) * T::SC;
#pragma unroll
        for (int c = 0; c < T::LS; ++c) {
            const uint32_t w = min(wave + c * T::NW, (uint32_t)T::BM / 64);
            const bool of_b = w == T::BM / 64;
            pipe::copy16_buf_asm(of_b ? rsb : rsa, to + w * (64 * 4 * T::G),
                                 (((of_b ? 0 : w * 64) + lane) * KB + grp * T::G) * 4);
        }
    };

    const uint32_t sw = pipe::swz<8>(row), o0 = (2 * q ^ sw) * 16, o1 = ((2 * q + 1) ^ sw) * 16;
    // Rows 16 i .. of a wave's operand: the permutation's second half differs by 16 rows.
    auto frag = [&](const uint8_t *base, int i) __attribute__((always_inline)) {
        const uint32_t flip = (i & 1) ? 2 * 16 : 0;   // swz<8>(r + 16) = swz<8>(r) ^ 2
        const uint8_t *p = base + (16 * i + row) * 128;
        return join(*reinterpret_cast<const u32x4 *>(p + (o0 ^ flip)), *reinterpret_cast<const u32x4 *>(p + (o1 ^ flip)));
    };
    auto a_of = [&](uint32_t step) { return lds + (step % S) * T::STAGE + wm * (16 * TM * 128); };
    auto b_of = [&](uint32_t step) { return lds + (step % S) * T::STAGE + T::A_BYTES + wn * (16 * TN * 128); };

    f32x4 acc[TM][TN], part[PART + 1];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i <= PART; ++i) part[i] = f32x4{0, 0, 0, 0};
    constexpr int R = TM % 4 == 0 ? 4 : 2;   // activation fragments held: two rows are read ahead, or the row after next
    static_assert(TM % R == 0, "the ring of fragments keeps its place from stage to stage");
    i32x8 fa[R], fb[TN];
    float sa[TM], last = 0.0f;   // this stage's scales; the last row's of the stage before

    // The sums are held here: the compiler would move additions behind a branch.
    auto hold = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < TM; ++x)
#pragma unroll
            for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[x][j]));
    };
    auto read_scales = [&](uint32_t t) __attribute__((always_inline)) {
        const uint8_t *sc = lds + S * T::STAGE + (t / T::G & 1) * T::SC + t % T::G * 4;
        const float sb = *reinterpret_cast<const float *>(sc + 4 * T::G * (T::BM + wn * (16 * TN) / KBLK));
#pragma unroll
        for (int i = 0; i < TM; ++i)
            sa[i] = *reinterpret_cast<const float *>(sc + 4 * T::G * (wm * (16 * TM) + 16 * i + row)) * sb;
    };
    // Product (i, j) of a stage is begun, and the one PART before it scaled and added.
    auto product = [&](int i, int j, const i32x8 &f) __attribute__((always_inline)) {
        const int p = i * TN + j, d = p - PART, e = d < 0 ? TM * TN + d : d;
        part[p % (PART + 1)] =
            __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], f, f32x4{0, 0, 0, 0}, FB, FA, 0, 0, 0, 0);
        const float s = d < 0 ? last : sa[e / TN];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            acc[e / TN][e % TN][x] = fmaf(part[(p + 1) % (PART + 1)][x], s, acc[e / TN][e % TN][x]);
    };

    if constexpr (T::TURNS) {
        // The two halves of the tile's rows take turns, a wave of each on a SIMD: while one half's
        // products run, the other copies its rows of a later stage and reads the first fragments
        // of its next one, which together take as long. A phase ends at a barrier; the second
        // half runs one behind. The first half's products of stage t are phase 2 t, its turnover
        // 2 t + 1, the second's 2 t + 1 and 2 t + 2. Both halves have stage t's weight fragments
        // in registers by the end of phase 2 t, so in phase 2 t + 1 the first half puts its rows
        // and the weight codes of stage t + 2 into the slot, in phase 2 t + 2 the second its rows;
        // each has landed before its next products' phase ends.
        auto turnover = [&](uint32_t t) __attribute__((always_inline)) {
            last = sa[TM - 1];
            fa[0] = frag(a_of(t), 0);
            fa[1] = frag(a_of(t), 1);
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j] = frag(b_of(t), j);
            read_scales(t);
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
                    product(i, j, fa[i % R]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            hold();
        };
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = 0.0f;
        issue_scales(0);
        issue(0);
        issue(1);
        pipe::wait_vmcnt<0>();
        barrier();
        if (wm == 0) {
            turnover(0);
            barrier();
            for (uint32_t t = 0; t < KB; ++t) {
                products(t);
                pipe::wait_vmcnt<0>();
                barrier();
                if (t % T::G == 0 && t + T::G < KB) issue_scales(t / T::G + 1);
                issue_a(t + 2, wave * T::LA, la);
                issue_b(t + 2, wave * 2 * T::LB, std::integral_constant<int, 2 * T::LB>{});
                turnover(t + 1);
                barrier();
            }
            barrier();
        } else {
            barrier();
            turnover(0);
            barrier();
            for (uint32_t t = 0; t < KB; ++t) {
                products(t);
                pipe::wait_vmcnt<0>();
                barrier();
                if (t % T::G == 0 && t + T::G < KB) issue_scales(t / T::G + 1);
                issue_a(t + 2, wave * T::LA, la);
                turnover(t + 1);
                barrier();
            }
        }
    } else {
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (s == 0) issue_scales(0);
        issue(s);
    }
    pipe::wait_vmcnt<(S - 1) * T::LOADS>();
    pipe::lds_barrier();
    fa[0] = frag(a_of(0), 0);
    fa[1] = frag(a_of(0), 1);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = frag(b_of(0), j);

    for (uint32_t t = 0; t < KB; ++t) {
        read_scales(t);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if (R == 4 && i + 2 < TM) fa[(i + 2) % R] = frag(a_of(t), i + 2);
            if (i == TM - 2) {
                // Every fragment and scale of this stage is in registers, and the next stage has
                // landed: behind the barrier its slot is read and this stage's is written.
                pipe::wait_lgkm0();
                pipe::wait_vmcnt<(S - 2) * T::LOADS>();
                pipe::lds_barrier();
                issue(t + S);
                // Every fourth stage the next four's scales. The sums are held here: the compiler
                // would move additions behind the branch.
                hold();
                if (t % T::G == 0 && t + T::G < KB) issue_scales(t / T::G + 1);
            }
            if (R == 4 && i >= TM - 2) fa[(i + 2) % R] = frag(a_of(t + 1), i + 2 - TM);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                product(i, j, fa[i % R]);
                if (i == TM - 1) fb[j] = frag(b_of(t + 1), j);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (R == 2) fa[i % R] = i + 2 < TM ? frag(a_of(t), i + 2) : frag(a_of(t + 1), i + 2 - TM);
        }
        last = sa[TM - 1];
    }
    }
    // The products still to be added.
#pragma unroll
    for (int e = TM * TN - PART; e < TM * TN; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            acc[e / TN][e % TN][x] = fmaf(part[e % (PART + 1)][x], last, acc[e / TN][e % TN][x]);
    static_assert((TM * TN) % (PART + 1) == 0 && PART <= TN, "the parts' ring keeps its place from stage to stage");

    pipe::wait_vmcnt<0>();   // the copies past the last stage, before LDS holds outputs

    // Epilogue through LDS: a lane holds four consecutive columns of a row; the workgroup
    // stores whole row segments.
    __syncthreads();
    constexpr uint32_t RB = T::BN * 2 + 16;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const f32x4 v = acc[i][j];
            *reinterpret_cast<u32x2 *>(lds + (wm * (16 * TM) + 16 * i + row) * RB + 2 * (wn * (16 * TN) + 16 * j + 4 * q)) =
                u32x2{f32_to_bf16_bits(v.x) | (f32_to_bf16_bits(v.y) << 16),
                      f32_to_bf16_bits(v.z) | (f32_to_bf16_bits(v.w) << 16)};
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

template <int FA, int FB, typename T>
int launch_tiles(const BlockArgs &g, hipStream_t st) {
    const uint32_t tiles_m = (g.M + T::BM - 1) / T::BM, tiles_n = (g.N + T::BN - 1) / T::BN, tiles = tiles_m * tiles_n;
    RENG_REQUIRE((uint64_t)tiles_m * tiles_n * (64 * T::NW) < (1ull << 32), "%u x %u outputs are too many for a launch", g.M,
                 g.N);
    hipLaunchKernelGGL((gemm_blocks_tiles<FA, FB, T>), dim3(tiles), dim3(64 * T::NW), T::LDS, st, g, tiles_m, tiles,
                       wide_mapm(tiles_m, tiles_n, T::BM, T::BN));
    return check_launch("gemm_blocks_tiles");
}

using Tile256 = BlockTile<8, 4, 2, 4, 2>;
using Tile128 = BlockTile<4, 4, 2, 2, 2>;
using Tile64 = BlockTile<2, 4, 2, 1, 3>;
static_assert(Tile256::BM == 256 && Tile256::BN == 256 && Tile128::BM == 128 && Tile128::BN == 128 &&
                  Tile64::BM == 64 && Tile64::BN == 64,
              "BLOCK_COST's tiles");

template <int FA, int FB>
int launch_blocks(const BlockArgs &g, hipStream_t st) {
    switch (block_pick(g.M, g.N, g.K, (uint64_t)device_props().cus)) {
    case BLK_RING_1x1: return launch_ring<FA, FB, 1, 1, 4, 4>(g, st);
    case BLK_RING_1x4: return launch_ring<FA, FB, 1, 4, 4, 2>(g, st);
    case BLK_RING_2x1: return launch_ring<FA, FB, 2, 1, 4, 3>(g, st);
    case BLK_RING_2x2: return launch_ring<FA, FB, 2, 2, 4, 2>(g, st);
    case BLK_RING_4x1: return launch_ring<FA, FB, 4, 1, 4, 2>(g, st);
    case BLK_RING_4x2: return launch_ring<FA, FB, 4, 2, 4, 2>(g, st);
    case BLK_RING_4x4: return launch_ring<FA, FB, 4, 4, 4, 2>(g, st);
    case BLK_TILE_64: return launch_tiles<FA, FB, Tile64>(g, st);
    case BLK_TILE_128: return launch_tiles<FA, FB, Tile128>(g, st);
    default: return launch_tiles<FA, FB, Tile256>(g, st);
    }
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
    // Offsets within a tile's 256 rows are 31 bits.
    RENG_REQUIRE(M <= 0x7fffffff && N <= 0x7fffffff && K <= (1u << 22), "dimension too large");
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
