// Grouped product of 8-bit operands, D_e = A_e B_e^T, in the block format of fp8_parts.h: tiles of 256 x 256 by v_mfma_scale_f32_16x16x128_f8f6f4,
// which multiplies 128 elements of reduction at a time (one block) and applies both operands' scales, fp32 sums throughout.
//
//  * A K step is one block of 128: 32 KB of each operand, brought into one of two LDS stages by direct global -> LDS loads (addresses are a
//    descriptor in scalar registers, one lane offset and a scalar offset; rows and columns past the end arrive as zeros). Eight wavefronts,
//    2 x 4, 128 x 64 each, 32 matrix instructions a step; their operands are two 16-byte LDS reads per 16 rows. The instruction wants 32
//    consecutive k a lane; both operands are given the same permutation of the block's k instead (bytes 16 q and 64 + 16 q), which leaves
//    every sum what it is and makes the reads free of bank conflicts.
//  * The 16 rows of B that make a fragment are not neighbours but rows 8 a + b (a, b = 0 .. 3) and, in the next fragment, 8 a + 4 + b:
//    a lane's results of two fragments are then eight neighbouring columns: 16 bytes of a 16-bit result, 8 of an 8-bit one.
//  * The loads are one stream over the steps of all tiles of a workgroup, two steps ahead: the last two steps of a tile load the first
//    two of the next. They are written in assembly, so the compiler places no waits for them; the one wait of a step, in front of its
//    last sixteenth-row block, is written by hand, and behind it the step's own stage is free again.
//  * Scales: a dword of four blocks per row of A (and per 128 rows of B) goes to LDS the same way every fourth step.
//  * Tall tiles (at most 256 groups): a tile may have 288 rows, 256 and one more row block per wavefront, whose 4 KB a step have stages of
//    their own.
//  * A reduction may be cut into segments (the two halves of a pre-activation): blocks begin anew in each.
//  * The instruction's sums: eight neighbouring products are aligned to the largest of them and cut below 2^-13 of it before they are added
//    to the fp32 sum (measured; the unscaled 8-bit instructions do the same), 2^-16 of a sum of random terms, root mean square. A result
//    that leaves in 16 bits loses nothing by that, and where a result becomes e4m3 the next product's many terms average the roundings that
//    fall to the other side (0.003 of the result instead of 0.0017; exact sums for a prefill's activation: 4096 tokens, hidden 2048, I 1408, E 64,
//    k 8, 356 -> 504 us, hidden 4096, I 14336, E 8, k 2, 1286 -> 1900). The pre-activation of a training pass, of which gradients are made
//    element by element, takes the bfloat16 instruction instead (k_step_exact).
//  * GLU: the tile holds 128 "up" and 128 "gate" columns; the activation, 128 columns or one block, is quantised from the fp32 sums: the
//    largest magnitude of a row goes from wavefront to wavefront through LDS. With KEEP the pre-activation is kept in 8 bits too.
//  * GLU_BWD: the product is the gradient of the activation; the pre-activation's gradient leaves, once rounded to 16 bits for the weight
//    gradient and once, from the unrounded values, in 8 bits for the input gradient.
#pragma once

#include "fp8_parts.h"
#include "gemm_parts.h"

namespace fmahip {
namespace fp8 {

using ::fmahip::gemm::kOutOfRange;
using ::fmahip::gemm::lds_address;
using ::fmahip::gemm::make_rsrc_words;
using ::fmahip::gemm::u32x4;
using ::fmahip::gemm::uniform;
using ::fmahip::gemm::wait_lds;
using ::fmahip::gemm::wait_vm;

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(8))) int i32x8;

constexpr int kTileM = 256, kTileN = 256;
constexpr int kWavesM = 2, kWavesN = 4, kWaves = kWavesM * kWavesN, kGemmThreads = kWaves * 64;
constexpr int kRowBlocks = 8, kColBlocks = 4;  // 16 x 16 blocks of a wavefront's 128 x 64
constexpr uint32_t kOperandBytes = 256 * kBlock, kStage = 2 * kOperandBytes;
constexpr int kTallM = 288;               // rows of a tall tile: 256, and one more row block per wavefront
constexpr uint32_t kTallGroups = 256;     // groups that a launch of the kernels for tall tiles may have (their table leaves room for the rows)
constexpr uint32_t kMaxGroups = FMA_MAX_GROUPS;

enum Epilogue { EPI_BF16, EPI_F16, EPI_F32, EPI_GLU, EPI_GLU_KEEP, EPI_GLU_BWD_BF16, EPI_GLU_BWD_F16 };

struct GemmArgs {
    const uint8_t *A, *A_s, *B, *B_s;
    const uint32_t* sizes;      // [E] rows per group; NULL: one group of R rows
    const int32_t* row_index;   // GLU: row i of A is row row_index[i] / divisor of a_rows
    uint32_t divisor, a_rows;
    uint32_t E, R, N, K, segs;  // K: elements of a segment of the reduction
    uint32_t a_pitch, a_seg, as_pitch, as_seg;            // bytes from row to row, from segment to segment
    uint32_t b_seg, bs_pitch, bs_seg, b_half, bs_half;    // half: from an expert's "up" matrix to its "gate" matrix
    uint64_t b_group, bs_group;
    void* D;                    // plain: [R, N]; GLU_BWD: [R, 2 N], the pre-activation's gradient
    uint8_t *out, *out_s;       // GLU: activation [R, N]; GLU_BWD: the pre-activation's gradient [R, 2, N]
    uint8_t *h, *h_s;           // pre-activation [R, 2, N]: written by GLU_KEEP, read by GLU_BWD
    uint32_t o_pitch_s;         // bytes of scales of N elements
};

__device__ __forceinline__ void load_lds16(u32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
    ::fmahip::gemm::buffer_load_lds_quiet(rsrc, voff, soff, lds);
}
__device__ __forceinline__ void fence_lds() { asm volatile("" ::: "memory"); }
// every LDS access of the workgroup in front of it is done (global stores stay in flight)
__device__ __forceinline__ void lds_barrier() {
    wait_lds();
    __builtin_amdgcn_s_barrier();
    fence_lds();
}
__device__ __forceinline__ u32x4 rsrc_at(uint64_t base, uint32_t bytes) {
    return u32x4{(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, bytes, 0x00020000u};
}
// everything from `base` on, for stores whose lanes have been checked (one that has nothing to store takes kOutOfRange)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(uint64_t base) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)base, 0, (int)0x7fffffff, 0x00020000);
}
__device__ __forceinline__ uint64_t uniform64(uint64_t x) { return ((uint64_t)uniform((uint32_t)(x >> 32)) << 32) | uniform((uint32_t)x); }

// two floats rounded to T, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (std::is_same_v<T, bf16_t>) return ::fmahip::gemm::ElemBf16::pack2(lo, hi);
    else return ::fmahip::gemm::ElemF16::pack2(lo, hi);
}

template <int EPI, bool TALL>
__global__ __launch_bounds__(kGemmThreads) void fp8_gemm_kernel(const GemmArgs args) {
    constexpr bool kGlu = EPI == EPI_GLU || EPI == EPI_GLU_KEEP;
    constexpr bool kBwd = EPI == EPI_GLU_BWD_BF16 || EPI == EPI_GLU_BWD_F16;
    constexpr bool kGather = kGlu;  // rows of A by index
    constexpr uint32_t kCols = kGlu ? kTileN / 2 : kTileN;  // columns of the output grid per tile
    constexpr bool kExact = EPI == EPI_GLU_KEEP;  // sums of exact products (k_step_exact)
    // Stores of an epilogue per wavefront, at least (0, 59: an epilogue that has waited for all loads in front of them itself)
    constexpr int kStores = EPI == EPI_BF16 || EPI == EPI_F16 ? 2 * kRowBlocks : (EPI == EPI_GLU ? kRowBlocks : (EPI == EPI_GLU_KEEP ? 3 * kRowBlocks : (kBwd ? 59 : 0)));
    constexpr uint32_t kMostGroups = TALL ? kTallGroups : kMaxGroups;
    constexpr int kBlocks = TALL ? kRowBlocks + 1 : kRowBlocks;  // row blocks of a wavefront, at most
    constexpr uint32_t kMostRows = TALL ? kTallM : kTileM;
    // per buffer: the scales of 256 rows of A, of two blocks of B (with the rest of that wavefront's load), and of the rows past 256
    constexpr uint32_t kScaleWords = TALL ? 384 : 320;
    constexpr int kMaxima = EPI == EPI_GLU_KEEP ? 3 : (kGlu ? 1 : (kBwd ? 1 : 0));

    __shared__ __attribute__((aligned(1024))) uint8_t s_op[2 * kStage];
    __shared__ __attribute__((aligned(256))) uint32_t s_scale[2 * kScaleWords];
    __shared__ __attribute__((aligned(16))) uint32_t s_max[kMaxima ? kMaxima * kMostRows * 4 : 4];
    __shared__ __attribute__((aligned(1024))) uint8_t s_x[TALL ? 2 * 32 * kBlock : 16];  // rows 256 .. 287 of A, per stage
    __shared__ __attribute__((aligned(1024))) uint8_t s_out[EPI == EPI_BF16 || EPI == EPI_F16 ? kWaves * 2048 : 16];
    __shared__ uint32_t s_tiles[kMostGroups + 1];  // row tiles of the groups before
    __shared__ uint32_t s_first[kMostGroups + 1];  // first row of the group

    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = uniform(tid >> 6);
    const uint32_t wm = wave / kWavesN, wn = wave % kWavesN;
    const uint32_t r16 = lane & 15u, q = lane >> 4;
    const uint32_t E = args.E, N = args.N, K = args.K;

    // ---- group table: rows past R do not exist, whatever the sizes say ----
    if (wave == 0) {
        uint32_t tiles = 0, rows = 0, height = kTileM;
        if constexpr (TALL) {
            // Tiles of up to 288 rows where they save more rounds of tiles than their longer steps cost, a tenth: experts of 256 or 512 +- 20 rows,
            // as an even routing makes them, otherwise pay a nearly empty tile every other time.
            uint32_t low = 0, high = 0;
            for (uint32_t e = lane; e < E; e += 64) {
                uint32_t m = args.sizes ? args.sizes[e] : args.R;
                m = m < args.R ? m : args.R;
                low += (m + kTileM - 1) / kTileM;
                high += (m + kTallM - 1) / kTallM;
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) {
                low += (uint32_t)__shfl_xor((int)low, d, 64);
                high += (uint32_t)__shfl_xor((int)high, d, 64);
            }
            const uint64_t columns = (N + kCols - 1) / kCols, g = gridDim.x;
            if ((high * columns + g - 1) / g * 11u < (low * columns + g - 1) / g * 10u) height = kTallM;
        }
        for (uint32_t base = 0; base < E; base += 64) {
            const uint32_t e = base + lane;
            uint32_t m = e < E ? (args.sizes ? args.sizes[e] : args.R) : 0u;
            m = m < args.R ? m : args.R;
            // (sums of 64 values of at most R fit 64 bits; what counts is clamped to R)
            const uint64_t end = rows + wave_inclusive_scan<uint64_t>(m);
            const uint32_t last = end < args.R ? (uint32_t)end : args.R;
            const uint64_t before = end - m;
            const uint32_t first = before < args.R ? (uint32_t)before : args.R;
            const uint32_t t = (last - first + height - 1) / height;
            const uint32_t it = wave_inclusive_scan<uint32_t>(t);
            if (e < E) {
                s_tiles[e] = tiles + it - t;
                s_first[e] = first;
            }
            tiles += __shfl(it, 63, 64);
            rows = __shfl(last, 63, 64);
        }
        if (lane == 0) {
            s_tiles[E] = tiles;
            s_first[E] = rows;
        }
    }
    __syncthreads();
    const uint32_t col_tiles = (N + kCols - 1) / kCols;
    const uint32_t total = uniform(s_tiles[E]) * col_tiles;
    const uint32_t grid = gridDim.x, per_xcd = grid / 8u;
    const uint32_t slot = grid % 8u == 0 ? (blockIdx.x % 8u) * per_xcd + blockIdx.x / 8u : blockIdx.x;
    if (slot >= total) return;

    const uint32_t k_blocks = (K + kBlock - 1) / kBlock;
    const uint32_t steps = k_blocks * args.segs;

    struct Tile {
        uint32_t e, row0, rows, n0;  // group, first packed row, rows, first column
    };
    // tile t (below `total`) of the sequence: a group's tiles one after the other, in blocks of eight row tiles, column by column
    auto find = [&](uint32_t t) -> Tile {
        const uint32_t row_tile = t / col_tiles;
        uint32_t e = 0;
        for (uint32_t base = 0; base < E; base += 64) {
            const bool before = base + lane < E && s_tiles[base + lane + 1] <= row_tile;
            const uint32_t n = (uint32_t)__popcll(__ballot(before));
            e += n;
            if (n < 64) break;
        }
        e = uniform(e);
        const uint32_t t0 = uniform(s_tiles[e]), mt = uniform(s_tiles[e + 1]) - t0;
        const uint32_t first = uniform(s_first[e]), end = uniform(s_first[e + 1]);
        const uint32_t in = t - t0 * col_tiles;
        const uint32_t block = in / (8u * col_tiles), at = in - block * 8u * col_tiles;
        const uint32_t height = mt - block * 8u < 8u ? mt - block * 8u : 8u;
        const uint32_t n = at / height, m = block * 8u + at - n * height;
        Tile tile;
        tile.e = e;
        tile.row0 = first + m * kTileM;
        uint32_t most = kTileM;
        if constexpr (TALL) {  // of a group's tiles as few as its rows need are tall, the first ones
            const uint32_t group = end - first, past = group > mt * kTileM ? (group - mt * kTileM + 31u) / 32u : 0u;
            tile.row0 += 32u * (m < past ? m : past);
            most += m < past ? 32u : 0u;
        }
        tile.rows = end - tile.row0 < most ? end - tile.row0 : most;
        tile.n0 = n * kCols;
        return tile;
    };

    // ---- the load stream ----
    const uint32_t lr = lane >> 3, lp = lane & 7u;
    uint32_t a_chunk = (lp ^ (((wave * 8u + lr) >> 1) & 7u)) * 16u;
    uint32_t b_chunk = (lp ^ ((wave & 3u) * 2u + ((lr >> 1) & 1u))) * 16u;
    uint32_t a_lane = (wave * 8u + lr) * args.a_pitch + a_chunk;
    uint32_t b_lane = (wave * 8u + lr) * K + b_chunk;
    const uint32_t lds0 = lds_address(s_op);
    const uint32_t lds_x = lds_address(s_x);
    const uint32_t lds_scale = lds_address(reinterpret_cast<const uint8_t*>(s_scale)) + wave * 256u;
    uint32_t l_tile = slot, l_ks = 0, l_seg = 0, l_stage = 0, l_quad = 0;  // next step to be loaded
    uint64_t l_a = 0, l_b = 0, l_b2 = 0, l_s = 0;  // addresses of the operands and of this wavefront's scales, at the current segment
    uint32_t l_a_bytes = 0, l_b_bytes = 0;
    constexpr int kGathered = TALL ? 5 : 4;
    uint32_t l_gather[kGathered] = {};
    uint32_t l_scale = kOutOfRange;  // this lane's offset into the scales
    Tile l_found = {0u, 0u, 0u, 0u};  // the tile that the loads are in
    auto aim = [&]() {
        if (l_tile >= total) {
            l_a_bytes = l_b_bytes = 0;
            l_scale = kOutOfRange;
            if constexpr (kGather) {
#pragma unroll
                for (int i = 0; i < kGathered; ++i) l_gather[i] = kOutOfRange;
            }
            return;
        }
        const Tile t = find(l_tile);
        l_found = t;
        const uint32_t n_block = t.n0 / kBlock;
        l_b = uniform64((uint64_t)(uintptr_t)args.B + t.e * args.b_group + (uint64_t)t.n0 * K);
        const uint32_t cols = N - t.n0 < kCols ? N - t.n0 : kCols;
        l_b_bytes = uniform(cols * K);
        if constexpr (kGlu) l_b2 = uniform64(l_b + args.b_half);
        if constexpr (kGather) {
            l_a = uniform64((uint64_t)(uintptr_t)args.A);
            l_a_bytes = args.a_rows * args.a_pitch;
#pragma unroll
            for (int i = 0; i < kGathered; ++i) {
                const uint32_t r = i * 64u + wave * 8u + lr;  // (i == 4: four wavefronts load rows 256 .. 287)
                const uint32_t src = r < t.rows ? (uint32_t)args.row_index[t.row0 + r] / args.divisor : args.a_rows;
                l_gather[i] = src < args.a_rows ? src * args.a_pitch + a_chunk : kOutOfRange;
            }
        } else {
            l_a = uniform64((uint64_t)(uintptr_t)args.A + (uint64_t)t.row0 * args.a_pitch);
            l_a_bytes = uniform(t.rows * args.a_pitch);
        }
        if (wave < 4 || (TALL && wave == 5)) {
            const uint32_t r = wave < 4 ? wave * 64u + lane : 256u + lane;
            l_s = (uint64_t)(uintptr_t)args.A_s;
            if constexpr (kGather) {
                const uint32_t src = r < t.rows ? (uint32_t)args.row_index[t.row0 + r] / args.divisor : args.a_rows;
                l_scale = src < args.a_rows ? src * args.as_pitch : kOutOfRange;
            } else {
                l_s += (uint64_t)t.row0 * args.as_pitch;
                l_scale = r < t.rows ? r * args.as_pitch : kOutOfRange;
            }
        } else {
            l_s = (uint64_t)(uintptr_t)args.B_s + t.e * args.bs_group + (uint64_t)n_block * args.bs_pitch;
            l_scale = lane == 0 ? 0u : kOutOfRange;
            if constexpr (kGlu) {
                if (lane == 1) l_scale = args.bs_half;
            } else {
                if (lane == 1 && t.n0 + kBlock < N) l_scale = args.bs_pitch;
            }
        }
        l_s = uniform64(l_s);
    };
    auto load_a = [&](int i) {
        uint32_t v = kGather ? l_gather[i] : a_lane;
        if (l_ks * kBlock + a_chunk >= K) v = kOutOfRange;
        load_lds16(rsrc_at(l_a, l_a_bytes), v, (kGather ? 0u : (uint32_t)i * 64u * args.a_pitch) + l_ks * kBlock,
                   lds0 + l_stage + ((uint32_t)i * 8u + wave) * 1024u);
    };
    auto load_b = [&](int i) {
        const uint32_t v = l_ks * kBlock + b_chunk >= K ? kOutOfRange : b_lane;
        const uint32_t rows = kGlu ? (uint32_t)(i & 1) * 64u : (uint32_t)i * 64u;
        load_lds16(rsrc_at(kGlu && i >= 2 ? l_b2 : l_b, l_b_bytes), v, rows * K + l_ks * kBlock,
                   lds0 + l_stage + kOperandBytes + ((uint32_t)i * 8u + wave) * 1024u);
    };
    auto load_x = [&]() {  // rows past 256, where the tile has any
        if constexpr (TALL) {
            if (l_found.rows > (uint32_t)kTileM && wave < 4) {
                uint32_t v = kGather ? l_gather[kGathered - 1] : a_lane;
                if (l_ks * kBlock + a_chunk >= K) v = kOutOfRange;
                load_lds16(rsrc_at(l_a, l_a_bytes), v, (kGather ? 0u : 256u * args.a_pitch) + l_ks * kBlock, lds_x + (l_stage ? 32u * kBlock : 0u) + wave * 1024u);
            }
        }
    };
    auto load_scales = [&]() {  // at the first of four steps
        if ((l_ks & 3u) == 0 && wave < (TALL ? 6u : 5u))
            ::fmahip::gemm::buffer_load_lds_quiet_b32(rsrc_at(l_s, 0x7fffffffu), l_scale, l_ks, lds_scale + l_quad * (kScaleWords * 4u));
    };
    auto next_load = [&]() {
        l_stage ^= kStage;
        ++l_ks;
        if (l_ks == k_blocks) {
            l_ks = 0;
            ++l_seg;
            if (l_seg == args.segs) {
                l_seg = 0;
                l_tile += grid;
                aim();
            } else {
                l_a += args.a_seg;
                l_b += args.b_seg;
                l_s += wave < 4 || (TALL && wave == 5) ? args.as_seg : args.bs_seg;
            }
        }
        if ((l_ks & 3u) == 0) l_quad ^= 1u;
    };

    // ---- fragments ----
    const uint32_t a_key = (r16 >> 1) & 7u, b_key = (r16 >> 2) * 2u + ((r16 >> 1) & 1u);
    uint32_t a_off = (wm * 128u + r16) * kBlock + ((q ^ a_key) << 4);
    const uint32_t b_base = kGlu ? wn * 32u : wn * 64u;
    uint32_t b_off = kOperandBytes + (b_base + (r16 >> 2) * 8u + (r16 & 3u)) * kBlock + ((q ^ b_key) << 4);
    // bytes from fragment 0 of B to fragment j
    auto b_step = [](int j) -> uint32_t { return (uint32_t)((kGlu ? (j >> 1) * 128 : (j >> 1) * 32) + (j & 1) * 4) * kBlock; };
    const uint8_t* const sc = reinterpret_cast<const uint8_t*>(s_scale);
    uint32_t sa_off = (wm * 128u + r16) * 4u;
    const uint32_t sb_off = (256u + (kGlu ? 0u : wn >> 1)) * 4u;
    uint32_t c_stage = 0, c_ks = 0, c_quad = 0;  // the step whose fragments are read

    auto read_frag = [&](uint32_t off) -> i32x8 {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(s_op + (c_stage + off));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(s_op + (c_stage + (off ^ 64u)));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto read_scale = [&](uint32_t off) -> int { return (int)sc[c_quad * (kScaleWords * 4u) + off + (c_ks & 3u)]; };

    // A row block's results are one 16-register value: the instruction's 4-register form has no variant whose result stays in place, and
    // without the value being named after every instruction results wander through the register file until it spills.
    f32x16 acc[kBlocks];
    i32x8 fa[2], fb[kColBlocks];
    int sa[2], sb[2];
    auto read_a = [&](int i, int buf) {
        fa[buf] = read_frag(a_off + (uint32_t)i * 16u * kBlock);
        sa[buf] = read_scale(sa_off + (uint32_t)i * 64u);
    };
    auto read_x = [&]() {  // the row block past 256, where block 6 was
        const uint32_t off = (c_stage ? 32u * kBlock : 0u) + (wm * 16u + r16) * kBlock + ((q ^ a_key) << 4);
        const i32x4 lo = *reinterpret_cast<const i32x4*>(s_x + off), hi = *reinterpret_cast<const i32x4*>(s_x + (off ^ 64u));
        fa[0] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        sa[0] = read_scale((320u + wm * 16u + r16) * 4u);
    };
    auto read_b = [&](int j) { fb[j] = read_frag(b_off + b_step(j)); };
    auto read_sb = [&]() {
        sb[0] = read_scale(sb_off);
        sb[1] = kGlu ? read_scale(sb_off + 4u) : sb[0];
    };
    i32x4 ha[2];  // (a training pass's products: half of A's fragment, bytes h * 64 on)
    auto read_half = [&](int h, int i, int buf) {
        ha[buf] = *reinterpret_cast<const i32x4*>(s_op + (c_stage + ((a_off + (uint32_t)i * 16u * kBlock) ^ (h ? 64u : 0u))));
        sa[buf] = read_scale(sa_off + (uint32_t)i * 64u);
    };
    auto read_half_x = [&](int h) {
        const uint32_t off = (c_stage ? 32u * kBlock : 0u) + (wm * 16u + r16) * kBlock + ((q ^ a_key) << 4);
        ha[0] = *reinterpret_cast<const i32x4*>(s_x + (off ^ (h ? 64u : 0u)));
        sa[0] = read_scale((320u + wm * 16u + r16) * 4u);
    };
    auto mma_with = [&](auto first_c, f32x16& c, int j, i32x8 a, int scale_a, int scale_b) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};  // (a tile's first step: the instruction takes the constant)
        if constexpr (!decltype(first_c)::value) v = f32x4{c[4 * j], c[4 * j + 1], c[4 * j + 2], c[4 * j + 3]};
        v = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], a, v, 0, 0, 0, scale_b, 0, scale_a);
        c[4 * j] = v[0];
        c[4 * j + 1] = v[1];
        c[4 * j + 2] = v[2];
        c[4 * j + 3] = v[3];
        asm("" : "+v"(c));
    };
    auto mma = [&](auto first_c, int i, int j, int buf, int scale_b) { mma_with(first_c, acc[i], j, fa[buf], sa[buf], scale_b); };
    auto next_step = [&]() {  // of the fragments
        c_stage ^= kStage;
        ++c_ks;
        if (c_ks == k_blocks) c_ks = 0;
        if ((c_ks & 3u) == 0) c_quad ^= 1u;
    };

    // ---- the first two steps ----
    aim();
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load_b(i);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_a(i);
        load_x();
        load_scales();
        next_load();
    }
    wait_vm<0>();
    lds_barrier();
    auto first_fragments = [&]() {
        read_sb();
#pragma unroll
        for (int j = 0; j < kColBlocks; ++j) read_b(j);
        if constexpr (kExact) read_half(0, 0, 0);
        else read_a(0, 0);
    };
    first_fragments();

    // The K step of a training pass's up projection (GLU_KEEP), whose result is rounded to e4m3 before a gradient is made of it. The 8-bit
    // instruction's cut (2^-16 of a sum, root mean square) moves one rounding in 2000 by a whole step, an eighth of the value, and dh with it:
    // weight gradients of a few rows, or of rows that cancel, then hold elements that are off by their size (0.46 of the tensor's root mean
    // square was seen among sizes of 128 tokens and more). Here the operands become bfloat16 in registers, with their scales, which loses
    // nothing, and the bfloat16 instruction sums them to 2^-26: 0.07 at most among thirty sizes. It costs half the matrix rate:
    // 8192 tokens with 8 of 64 experts, 2048 x 1408, forward and backward take 3420 us instead of 3190. The gradient's product (GLU_BWD) has
    // its result rounded to e4m3 for the input's gradient alone, where a row's many columns average it: it would take 110 us more.
    // (Scaled values below bfloat16's smallest, 2^-133, are lost; their block's largest is below 2^-110.)
    // Half a step's K at a time, so that the converted fragments fit beside the sums: both halves of B stay raw until their turn.
    using gemm::bf16x8;
    using gemm::bf16x2;
    bf16x8 bx[kColBlocks][2], ax[2];
    auto widen = [](bf16x8 (&to)[2], const int* raw, int scale) {
        const float factor = __uint_as_float((uint32_t)scale << 23);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[2 * s + k], factor, false);
                const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[2 * s + k], factor, true);
                to[s][4 * k] = lo[0];
                to[s][4 * k + 1] = lo[1];
                to[s][4 * k + 2] = hi[0];
                to[s][4 * k + 3] = hi[1];
            }
        }
    };
    auto widen_b = [&](int h) {
#pragma unroll
        for (int j = 0; j < kColBlocks; ++j) {
            const int raw[4] = {fb[j][4 * h], fb[j][4 * h + 1], fb[j][4 * h + 2], fb[j][4 * h + 3]};
            widen(bx[j], raw, sb[j >> 1]);
        }
    };
    auto mma_half = [&](auto first_c, f32x16& c, int buf, auto&& between) {
        const int raw[4] = {ha[buf][0], ha[buf][1], ha[buf][2], ha[buf][3]};
        widen(ax, raw, sa[buf]);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int j = 0; j < kColBlocks; ++j) {
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
                if (s || !decltype(first_c)::value) v = f32x4{c[4 * j], c[4 * j + 1], c[4 * j + 2], c[4 * j + 3]};
                v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bx[j][s], ax[s], v, 0, 0, 0);
                c[4 * j] = v[0];
                c[4 * j + 1] = v[1];
                c[4 * j + 2] = v[2];
                c[4 * j + 3] = v[3];
                asm("" : "+v"(c));
                if (s == 1) between(j);
            }
        }
    };
    auto k_step_exact = [&](auto first_c, bool tall) {
        constexpr bool FIRST = decltype(first_c)::value;
        using Sum = std::integral_constant<bool, false>;
        const auto nothing = [](int) {};
        // (the loads and barriers of the step below, with the same reasons)
        widen_b(0);
#pragma unroll
        for (int i = 0; i < kRowBlocks; ++i) {
            if (i == 1) lds_barrier();
            if (i < kRowBlocks - 1) read_half(0, i + 1, (i + 1) & 1);
            if (i == 1) mma_half(first_c, acc[i], i & 1, [&](int j) { load_b(j); });
            else mma_half(first_c, acc[i], i & 1, nothing);
            if (i == kRowBlocks - 2) {
                if constexpr (TALL) {
                    if (tall) {
                        read_half_x(0);
                        mma_half(first_c, acc[kBlocks - 1], 0, nothing);
                    }
                }
                read_half(1, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        widen_b(1);
#pragma unroll
        for (int i = 0; i < kRowBlocks - 1; ++i) {
            read_half(1, i + 1, (i + 1) & 1);
            mma_half(Sum{}, acc[i], i & 1, nothing);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (TALL) {
            if (tall) {
                read_half_x(1);
                mma_half(Sum{}, acc[kBlocks - 1], 0, nothing);
            }
        }
        wait_vm<(FIRST ? (4 + kStores < 63 ? 4 + kStores : 63) : 4)>();
        lds_barrier();
        next_step();
        mma_half(Sum{}, acc[kRowBlocks - 1], (kRowBlocks - 1) & 1, [&](int j) {
            load_a(j);
            read_b(j);
        });
        read_sb();
        read_half(0, 0, 0);
        load_x();
        load_scales();
        next_load();
    };

    // One K step of a tile; FIRST: of its first, whose sums begin at zero.
    auto k_step = [&](auto first_c, bool tall) {
        constexpr bool FIRST = decltype(first_c)::value;
#pragma unroll
        for (int i = 0; i < kRowBlocks - 1; ++i) {
            // The step's fragments of B are in registers, in every wavefront (its first products have used them): the loads of B two steps
            // on may fill their place.
            if (i == 1) lds_barrier();
            read_a(i + 1, (i + 1) & 1);
#pragma unroll
            for (int j = 0; j < kColBlocks; ++j) {
                mma(first_c, i, j, i & 1, sb[j >> 1]);
                if (i == 1) load_b(j);
            }
            if (TALL && i == kRowBlocks - 2 && tall) read_x();
            __builtin_amdgcn_sched_barrier(0);
        }
        // Every fragment of the step is read, and the next step has landed (all but the loads of B just issued): the next step's fragments
        // are read from here on, and the loads of A two steps on fill this step's place. In a tile's first step the stores of the
        // epilogue before it are younger than what is waited for, and stay outstanding.
        wait_vm<(FIRST ? (4 + kStores < 63 ? 4 + kStores : 63) : 4)>();
        lds_barrier();
        next_step();
        {
            constexpr int i = kRowBlocks - 1;
            const int s0 = sb[0], s1 = sb[1];
            read_sb();
            if constexpr (TALL) {
                if (tall) {
#pragma unroll
                    for (int j = 0; j < kColBlocks; ++j) mma_with(first_c, acc[kBlocks - 1], j, fa[0], sa[0], j < 2 ? s0 : s1);
                }
            }
#pragma unroll
            for (int j = 0; j < kColBlocks; ++j) {
                mma(first_c, i, j, i & 1, j < 2 ? s0 : s1);
                load_a(j);
                read_b(j);
            }
            read_a(0, 0);
        }
        load_x();
        load_scales();
        next_load();
    };

    Tile t = l_found;
    for (uint32_t c_tile = slot; c_tile < total; c_tile += grid) {
        if (steps < 3) t = find(c_tile);  // (the loads are two steps ahead: with three and more they are in this tile when it begins)
        else t = l_found;
        const bool tall = TALL && t.rows > (uint32_t)kTileM;
        if constexpr (kExact) {
            k_step_exact(std::integral_constant<bool, true>{}, tall);
            for (uint32_t step = 1; step < steps; ++step) k_step_exact(std::integral_constant<bool, false>{}, tall);
        } else {
            k_step(std::integral_constant<bool, true>{}, tall);
            for (uint32_t step = 1; step < steps; ++step) k_step(std::integral_constant<bool, false>{}, tall);
        }
        // first row of this wavefront's row block i
        auto block_row = [&](int i) -> uint32_t { return i < kRowBlocks ? wm * 128u + (uint32_t)i * 16u : 256u + wm * 16u; };

        // ---- epilogue ----
        // (addresses that follow from the lane are computed here, anew for every tile: kept over the K loop they would be spilled)
        uint32_t here = lane;
        asm volatile("" : "+v"(here));
        {
        const uint32_t lane = here, r16 = lane & 15u, q = lane >> 4;
        if constexpr (EPI == EPI_BF16 || EPI == EPI_F16) {
            using T = std::conditional_t<EPI == EPI_BF16, bf16_t, f16_t>;
            uint16_t* const tile = (uint16_t*)args.D + (uint64_t)t.row0 * N + t.n0;
            if (N % 8u == 0) {
                // Through 2 KB of LDS per wavefront, 16 rows at a time, so that eight neighbouring lanes store a line of 128 bytes: straight from the
                // registers neighbouring lanes are in different rows, and a store takes as many turns of the address unit as it has lines.
                const __amdgpu_buffer_rsrc_t rsrc = ::fmahip::gemm::make_rsrc(tile, uniform(t.rows * N - t.n0) * 2u);
                uint8_t* const image = s_out + wave * 2048u;
                const uint32_t chunk = lane & 7u, line = lane >> 3;
                const uint32_t col = wn * 64u + chunk * 8u;
                const bool in = t.n0 + col < N;
                const uint32_t put = r16 * 128u + ((q ^ (r16 & 7u)) << 4), get = line * 128u + ((chunk ^ line) << 4);
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                if (i >= kRowBlocks && !tall) continue;
                    u32x4 v[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int x = 0; x < 4; ++x) v[p][x] = pack_pair<T>(acc[i][8 * p + 2 * x], acc[i][8 * p + 2 * x + 1]);
                    *reinterpret_cast<u32x4*>(image + put) = v[0];
                    *reinterpret_cast<u32x4*>(image + (put ^ 64u)) = v[1];
                    const u32x4 low = *reinterpret_cast<const u32x4*>(image + get), high = *reinterpret_cast<const u32x4*>(image + 1024u + get);
                    const uint32_t at = ((block_row(i) + line) * N + col) * 2u;
                    ::fmahip::gemm::store_tile16<false>(rsrc, in ? at : kOutOfRange, __builtin_bit_cast(uint4, low));
                    ::fmahip::gemm::store_tile16<false>(rsrc, in ? at + N * 16u : kOutOfRange, __builtin_bit_cast(uint4, high));
                }
            } else {
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                if (i >= kRowBlocks && !tall) continue;
                    const uint32_t row = block_row(i) + r16;
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const uint32_t col = wn * 64u + (uint32_t)(x / 8) * 32u + q * 8u + (uint32_t)(x % 8);
                        if (row < t.rows && t.n0 + col < N) tile[(uint64_t)row * N + col] = (uint16_t)pack_pair<T>(acc[i][x], 0.f);
                    }
                }
                wait_vm<0>();
            }
        } else if constexpr (EPI == EPI_F32) {
            float* const tile = (float*)args.D + (uint64_t)t.row0 * N + t.n0;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                if (i >= kRowBlocks && !tall) continue;
                const uint32_t row = block_row(i) + r16;
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    const uint32_t col = wn * 64u + (uint32_t)(x / 8) * 32u + q * 8u + (uint32_t)(x % 8);
                    float* const to = tile + (uint64_t)row * N + col;
                    if (row < t.rows) {
                        if (N % 4u == 0) {
                            if (t.n0 + col < N) *reinterpret_cast<f32x4*>(to) = f32x4{acc[i][x], acc[i][x + 1], acc[i][x + 2], acc[i][x + 3]};
                        } else {
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                if (t.n0 + col + y < N) to[y] = acc[i][x + y];
                        }
                    }
                }
            }
            wait_vm<0>();
        } else if constexpr (kGlu) {
            const uint32_t block = t.n0 / kBlock;
            // magnitudes of the row's columns of this wavefront
            auto row_max = [&](uint32_t m) -> uint32_t {
                m = max_u32(m, (uint32_t)__shfl_xor((int)m, 16, 64));
                return max_u32(m, (uint32_t)__shfl_xor((int)m, 32, 64));
            };
            // `what` 0: the activation, which has taken the place of the sums of "up" by then; 1, 2: the pre-activation's halves
            auto maxima = [&](int what) {
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    if (i >= kRowBlocks && !tall) continue;
                    uint32_t m = 0;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        if (what == 0) {
                            const float g = acc[i][8 + x];
                            acc[i][x] = acc[i][x] * g * sigmoid_clamped_fast(g);
                        }
                        m = max_u32(m, magnitude_bits(acc[i][(what == 2 ? 8 : 0) + x]));
                    }
                    m = row_max(m);
                    if (q == 0) s_max[((uint32_t)what * kMostRows + block_row(i) + r16) * 4u + wn] = m;
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            auto store = [&](int what) {
                asm volatile("" : "+v"(here));  // (as above, for every one of them)
                const uint32_t lane = here, r16 = lane & 15u, q = lane >> 4, col = t.n0 + wn * 32u + q * 8u;
                // values of this tile's rows (the rows' ends are looked at here), and their scales
                const uint32_t pitch = what == 0 ? N : 2u * N, s_pitch = what == 0 ? args.o_pitch_s : 2u * args.o_pitch_s;
                const uint64_t values = what == 0 ? (uint64_t)(uintptr_t)args.out + (uint64_t)t.row0 * pitch
                                                  : (uint64_t)(uintptr_t)args.h + (uint64_t)t.row0 * pitch + (what == 2 ? N : 0u);
                const uint64_t scales = what == 0 ? (uint64_t)(uintptr_t)args.out_s + (uint64_t)t.row0 * s_pitch
                                                  : (uint64_t)(uintptr_t)args.h_s + (uint64_t)t.row0 * s_pitch + (what == 2 ? args.o_pitch_s : 0u);
                const __amdgpu_buffer_rsrc_t rv = buffer_at(values), rs = buffer_at(scales);
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    if (i >= kRowBlocks && !tall) continue;
                    const uint32_t row = block_row(i) + r16;
                    const uint4 m = *reinterpret_cast<const uint4*>(s_max + ((uint32_t)what * kMostRows + row) * 4u);
                    const uint32_t byte = scale_byte(max_u32(max_u32(m.x, m.y), max_u32(m.z, m.w)));
                    const float inverse = scale_inverse(byte);
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = acc[i][(what == 2 ? 8 : 0) + x] * inverse;
                    const u32x2 o = {pack4(v[0], v[1], v[2], v[3]), pack4(v[4], v[5], v[6], v[7])};
                    const bool live = row < t.rows;
                    __builtin_amdgcn_raw_buffer_store_b64(o, rv, (int)(live && col < N ? row * pitch + col : kOutOfRange), 0, 0);
                    if (wn == 0)
                        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)byte, rs, (int)(live && q == 0 ? row * s_pitch + block : kOutOfRange), 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if constexpr (EPI == EPI_GLU_KEEP) {
                maxima(1);
                maxima(2);
                lds_barrier();
                store(1);
                store(2);
            }
            maxima(0);
            lds_barrier();
            store(0);
        } else {
            using T = std::conditional_t<EPI == EPI_GLU_BWD_BF16, bf16_t, f16_t>;
            // columns of block wn / 2 of the tile's two
            const uint32_t block = t.n0 / kBlock + (wn >> 1);
            const uint32_t s_pitch = args.o_pitch_s;
            wait_vm<0>();
            // The pre-activation of a row block: eight columns of each half twice, and the scales, requested two blocks ahead. Loads and stores
            // are unconditional (a lane without work has an offset out of range): the compiler then counts them, and no block waits
            // for the stores of the one before.
            struct Kept {
                u32x2 v[2][2];  // [half][columns p]
                uint32_t s[2];
            };
            constexpr int kAhead = 2;
            Kept kept[kAhead];
            const bool in = t.n0 + (wn >> 1) * kBlock < N;
            const uint64_t first_value = (uint64_t)t.row0 * (2u * (uint64_t)N), first_scale = (uint64_t)t.row0 * (2u * s_pitch);
            const __amdgpu_buffer_rsrc_t r_h = buffer_at((uint64_t)(uintptr_t)args.h + first_value), r_hs = buffer_at((uint64_t)(uintptr_t)args.h_s + first_scale);
            const __amdgpu_buffer_rsrc_t r_d = buffer_at((uint64_t)(uintptr_t)args.D + 2u * first_value);
            const __amdgpu_buffer_rsrc_t r_o = buffer_at((uint64_t)(uintptr_t)args.out + first_value), r_os = buffer_at((uint64_t)(uintptr_t)args.out_s + first_scale);
            auto value_at = [&](uint32_t row, int h, int p) -> uint32_t {
                const uint32_t col = t.n0 + wn * 64u + (uint32_t)p * 32u + q * 8u;
                return row < t.rows && col < N ? row * 2u * N + (uint32_t)h * N + col : kOutOfRange;
            };
            auto scale_at = [&](uint32_t row, int h) -> uint32_t { return row < t.rows && in ? row * 2u * s_pitch + (uint32_t)h * s_pitch + block : kOutOfRange; };
            auto fetch = [&](int i) -> Kept {
                const uint32_t row = block_row(i) + r16;
                Kept k;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    k.s[h] = __builtin_amdgcn_raw_buffer_load_b8(r_hs, (int)scale_at(row, h), 0, 0);
#pragma unroll
                    for (int p = 0; p < 2; ++p) k.v[h][p] = __builtin_amdgcn_raw_buffer_load_b64(r_h, (int)value_at(row, h, p), 0, 0);
                }
                return k;
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) kept[i] = fetch(i);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                if (i >= kRowBlocks && !tall) continue;
                const uint32_t row = block_row(i) + r16;
                const Kept k = kept[i % kAhead];
                if (i + kAhead < kBlocks) kept[i % kAhead] = fetch(i + kAhead);
                float d[2][2][8];  // [half][columns p][x]
                uint32_t m[2] = {0u, 0u};
                const float su = finite_scale_value(k.s[0]), sg = finite_scale_value(k.s[1]);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float u[8], g[8];
                    unpack4(k.v[0][p][0], *reinterpret_cast<float(*)[4]>(u));
                    unpack4(k.v[0][p][1], *reinterpret_cast<float(*)[4]>(u + 4));
                    unpack4(k.v[1][p][0], *reinterpret_cast<float(*)[4]>(g));
                    unpack4(k.v[1][p][1], *reinterpret_cast<float(*)[4]>(g + 4));
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        swiglu_b<T>(g[x] * sg, u[x] * su, acc[i][8 * p + x], d[1][p][x], d[0][p][x]);
                        m[0] = max_u32(m[0], magnitude_bits(d[0][p][x]));
                        m[1] = max_u32(m[1], magnitude_bits(d[1][p][x]));
                    }
                }
                // the other wavefront of the block has its half of the row: slots alternate, so one barrier per row block is enough
                uint32_t* const slots = s_max + (uint32_t)(i & 1) * 256u;  // [wave][half][16]
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    m[h] = max_u32(m[h], (uint32_t)__shfl_xor((int)m[h], 16, 64));
                    m[h] = max_u32(m[h], (uint32_t)__shfl_xor((int)m[h], 32, 64));
                    if (q == 0) slots[(wave * 2u + (uint32_t)h) * 16u + r16] = m[h];
                }
                lds_barrier();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t byte = scale_byte(max_u32(m[h], slots[((wave ^ 1u) * 2u + (uint32_t)h) * 16u + r16]));
                    const float inverse = scale_inverse(byte);
                    __builtin_amdgcn_raw_buffer_store_b8((uint8_t)byte, r_os, (int)(q == 0 && (wn & 1u) == 0 ? scale_at(row, h) : kOutOfRange), 0, 0);
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const float(&v)[8] = d[h][p];
                        const uint32_t at = value_at(row, h, p);
                        const u32x4 o = {pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]), pack_pair<T>(v[4], v[5]), pack_pair<T>(v[6], v[7])};
                        ::fmahip::gemm::store_tile16<false>(r_d, at == kOutOfRange ? kOutOfRange : 2u * at, __builtin_bit_cast(uint4, o));
                        const u32x2 o8 = {pack4(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                                          pack4(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse)};
                        __builtin_amdgcn_raw_buffer_store_b64(o8, r_o, (int)at, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        }
        if constexpr (kBwd) {
            // What the loads and fragments take from the lane, formed anew: kept over this epilogue these registers were spilled, and their reloads
            // waited for the whole load stream in every K step (64 x 1024 rows, 1408 x 2048: 476 -> 425 us).
            asm volatile("" : "+v"(here));
            const uint32_t lr = here >> 3, lp = here & 7u, r16 = here & 15u, q = here >> 4;
            const uint32_t a_key = (r16 >> 1) & 7u, b_key = (r16 >> 2) * 2u + ((r16 >> 1) & 1u);
            a_chunk = (lp ^ (((wave * 8u + lr) >> 1) & 7u)) * 16u;
            b_chunk = (lp ^ ((wave & 3u) * 2u + ((lr >> 1) & 1u))) * 16u;
            a_lane = (wave * 8u + lr) * args.a_pitch + a_chunk;
            b_lane = (wave * 8u + lr) * K + b_chunk;
            a_off = (wm * 128u + r16) * kBlock + ((q ^ a_key) << 4);
            b_off = kOperandBytes + (b_base + (r16 >> 2) * 8u + (r16 & 3u)) * kBlock + ((q ^ b_key) << 4);
            sa_off = (wm * 128u + r16) * 4u;
        }
        // The next tile's first fragments once more: 42 registers that these epilogues use meanwhile.
        if constexpr (kGlu || kBwd) first_fragments();
    }
    wait_vm<0>();  // loads past the last step write zeros into LDS: they are done when the workgroup ends
}

}  // namespace fp8
}  // namespace fmahip
