// To the 8-bit block format and back (fp8_parts.h): HBM-bound element kernels.
//
// Rows: half a wavefront takes 512 neighbouring elements of a row, 16 a lane, so that a block of 128 is eight lanes (three exchanges for
// its largest magnitude), its values leave as 16 bytes a lane and the four scales as one dword. One-shot workgroups with all loads in
// front. [16384, 4096] bf16 35 us (5.8 TB/s); eight elements a lane 39, without the non-temporal hint 38.
// Weights: a workgroup takes one 128 x 128 block, eight by eight elements a thread; the transposed copy, which the input gradient's product
// reads along its own reduction, is made from the same registers through 17 KB of LDS, so that the 16-bit weights are read once. 64 matrices
// of 2816 x 2048, bf16, with the copy: 262 us (5.6 TB/s).
#include "fp8_parts.h"
#include "gemm_parts.h"

namespace fmahip {
namespace {
using namespace fp8;

constexpr int kThreads = 256;

template <typename T, int N>
__device__ __forceinline__ void load_floats(const T* p, float (&f)[N]) {
    constexpr int V = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < N / V; ++i) {
        const Vec16<T> v = load_streaming16(reinterpret_cast<const Vec16<T>*>(p) + i);
#pragma unroll
        for (int e = 0; e < V; ++e) f[i * V + e] = Num<T>::up(v.v[e]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* p, const float (&f)[N]) {
    constexpr int V = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < N / V; ++i) {
        Vec16<T> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = Num<T>::down(f[i * V + e]);
        Vec16<T>* const to = reinterpret_cast<Vec16<T>*>(p) + i;
        if constexpr (N == V) store_streaming16(to, v);
        else *to = v;
    }
}

// ---- rows -----------------------------------------------------------------------------------------------------------

// K a multiple of 16. `quads` of 512 elements per row; a workgroup takes UNROLL * 8 neighbouring quads, eight at a time
template <typename T, int UNROLL>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ values,
                                                                 uint32_t* __restrict__ scales, int64_t total, uint32_t quads,
                                                                 int64_t K) {
    const uint32_t lane = threadIdx.x & 31u;
    const int64_t first = (int64_t)blockIdx.x * (UNROLL * (kThreads / 32)) + threadIdx.x / 32;
    float f[UNROLL][16];
    int64_t at[UNROLL], unit[UNROLL];
    bool in[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        unit[u] = first + u * (kThreads / 32);
        const int64_t row = total < (1ll << 31) ? (int64_t)((uint32_t)unit[u] / quads) : unit[u] / quads;
        const int64_t k = (unit[u] - row * quads) * 512 + lane * 16;
        in[u] = unit[u] < total && k < K;
        at[u] = row * K + k;
        if (in[u]) {
            load_floats(x + at[u], f[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[u][i] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max_u32(m, magnitude_bits(f[u][i]));
        const uint32_t byte = scale_byte(group_max<8>(m));
        const float inverse = scale_inverse(byte);
        uint4 q;
        q.x = pack4(f[u][0] * inverse, f[u][1] * inverse, f[u][2] * inverse, f[u][3] * inverse);
        q.y = pack4(f[u][4] * inverse, f[u][5] * inverse, f[u][6] * inverse, f[u][7] * inverse);
        q.z = pack4(f[u][8] * inverse, f[u][9] * inverse, f[u][10] * inverse, f[u][11] * inverse);
        q.w = pack4(f[u][12] * inverse, f[u][13] * inverse, f[u][14] * inverse, f[u][15] * inverse);
        if (in[u]) *reinterpret_cast<uint4*>(values + at[u]) = q;
        // (a block's first lane is inside the row if the block has any element)
        uint32_t four = __shfl((int)in[u], (int)(threadIdx.x & 63u) & ~7, kWave) ? byte : 127u;
        four <<= (lane >> 3) * 8u;
        four |= (uint32_t)__shfl_xor((int)four, 8, kWave);
        four |= (uint32_t)__shfl_xor((int)four, 16, kWave);
        if (lane == 0 && unit[u] < total) scales[unit[u]] = four;
    }
}

// any K, any alignment: eight lanes per block, element by element
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_rows_generic_kernel(const T* __restrict__ x, uint8_t* __restrict__ values,
                                                                         uint8_t* __restrict__ scales, int64_t total, int64_t pitch,
                                                                         int64_t K) {
    const uint32_t lane = threadIdx.x & 7u;
    const int64_t step = (int64_t)gridDim.x * (kThreads / 8);
    // (every lane of a wavefront makes the same number of turns: the exchange below needs them all)
    for (int64_t base = (int64_t)blockIdx.x * (kThreads / 8); base < total; base += step) {
        const int64_t block = base + threadIdx.x / 8;
        const int64_t row = block / pitch, k0 = (block - row * pitch) * kBlock;
        const int64_t n = block < total && k0 < K ? (K - k0 < kBlock ? K - k0 : kBlock) : 0;
        const T* p = x + row * K + k0;
        uint32_t m = 0;
        for (int64_t i = lane; i < n; i += 8) m = max_u32(m, magnitude_bits(Num<T>::up(p[i])));
        const uint32_t byte = scale_byte(group_max<8>(m));
        const float inverse = scale_inverse(byte);
        for (int64_t i = lane; i < n; i += 8) values[row * K + k0 + i] = (uint8_t)pack4(Num<T>::up(p[i]) * inverse, 0.f, 0.f, 0.f);
        if (lane == 0 && block < total) scales[block] = (uint8_t)(n ? byte : 127u);
    }
}

// ---- 128 x 128 blocks -----------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* slot) {
    m = group_max<64>(m);
    if ((threadIdx.x & 63u) == 0) slot[threadIdx.x >> 6] = m;
    __syncthreads();
    return max_u32(max_u32(slot[0], slot[1]), max_u32(slot[2], slot[3]));
}

// The scale of block (n, k) of matrix e: byte k of row n of [n_blocks, pitch_k], and byte n of row k of the transposed [k_blocks, pitch_n];
// the last block of a row fills the row up to whole dwords.
__device__ __forceinline__ void store_block_scales(uint8_t* scales, uint8_t* scales_t, int64_t e, int64_t n, int64_t k, int64_t n_blocks,
                                                   int64_t k_blocks, uint32_t byte) {
    if (threadIdx.x < 4) {
        const int64_t pitch_k = (k_blocks + 3) & ~(int64_t)3, pitch_n = (n_blocks + 3) & ~(int64_t)3;
        const int64_t i = threadIdx.x;
        if (i == 0 || (k == k_blocks - 1 && k + i < pitch_k)) scales[(e * n_blocks + n) * pitch_k + k + i] = (uint8_t)(i ? 127u : byte);
        if (scales_t && (i == 0 || (n == n_blocks - 1 && n + i < pitch_n)))
            scales_t[(e * k_blocks + k) * pitch_n + n + i] = (uint8_t)(i ? 127u : byte);
    }
}

// K a multiple of 8, and N too with a transposed copy
template <typename T, bool TRANSPOSED>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(const T* __restrict__ x, uint8_t* __restrict__ values,
                                                                   uint8_t* __restrict__ scales, uint8_t* __restrict__ values_t,
                                                                   uint8_t* __restrict__ scales_t, int64_t N, int64_t K,
                                                                   uint32_t n_blocks, uint32_t k_blocks) {
    constexpr uint32_t kPitch = 136;  // bytes of a row of the transposed image: rows 34 banks apart
    __shared__ uint32_t s_max[4];
    __shared__ __attribute__((aligned(16))) uint8_t s_t[TRANSPOSED ? kBlock * kPitch : 16];
    const uint32_t k = blockIdx.x % k_blocks, en = blockIdx.x / k_blocks;
    const uint32_t n = en % n_blocks, e = en / n_blocks;
    const uint32_t pc = threadIdx.x & 15u, pr = threadIdx.x >> 4;  // this thread's eight by eight elements
    const int64_t col = (int64_t)k * kBlock + pc * 8, row = (int64_t)n * kBlock + pr * 8;
    const int64_t base = (int64_t)e * N * K;
    float f[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (row + i < N && col < K) {
            load_floats(x + base + (row + i) * K + col, f[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_u32(m, magnitude_bits(f[i][j]));
    const uint32_t byte = scale_byte(block_max(m, s_max));
    const float inverse = scale_inverse(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] *= inverse;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (row + i < N && col < K) {
            uint2 q;
            q.x = pack4(f[i][0], f[i][1], f[i][2], f[i][3]);
            q.y = pack4(f[i][4], f[i][5], f[i][6], f[i][7]);
            *reinterpret_cast<uint2*>(values + base + (row + i) * K + col) = q;
        }
    }
    if constexpr (TRANSPOSED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint2 q;
            q.x = pack4(f[0][j], f[1][j], f[2][j], f[3][j]);
            q.y = pack4(f[4][j], f[5][j], f[6][j], f[7][j]);
            *reinterpret_cast<uint2*>(s_t + (pc * 8 + j) * kPitch + pr * 8) = q;
        }
        __syncthreads();
        // rows of 128 bytes, 16 threads each
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t r = (uint32_t)i * 16u + pr;
            if ((int64_t)k * kBlock + r < K && (int64_t)n * kBlock + pc * 8 < N)
                *reinterpret_cast<uint2*>(values_t + base + ((int64_t)k * kBlock + r) * N + (int64_t)n * kBlock + pc * 8) =
                    *reinterpret_cast<const uint2*>(s_t + r * kPitch + pc * 8);
        }
    }
    store_block_scales(scales, scales_t, e, n, k, n_blocks, k_blocks, byte);
}

// any N and K: element by element
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_blocks_generic_kernel(const T* __restrict__ x, uint8_t* __restrict__ values,
                                                                           uint8_t* __restrict__ scales, uint8_t* __restrict__ values_t,
                                                                           uint8_t* __restrict__ scales_t, int64_t N, int64_t K,
                                                                           uint32_t n_blocks, uint32_t k_blocks) {
    __shared__ uint32_t s_max[4];
    const uint32_t k = blockIdx.x % k_blocks, en = blockIdx.x / k_blocks;
    const uint32_t n = en % n_blocks, e = en / n_blocks;
    const int64_t col0 = (int64_t)k * kBlock, row0 = (int64_t)n * kBlock, base = (int64_t)e * N * K;
    const int64_t cols = K - col0 < kBlock ? K - col0 : kBlock, rows = N - row0 < kBlock ? N - row0 : kBlock;
    uint32_t m = 0;
    for (int64_t i = threadIdx.x; i < rows * kBlock; i += kThreads) {
        const int64_t r = row0 + i / kBlock, c = i % kBlock;
        if (c < cols) m = max_u32(m, magnitude_bits(Num<T>::up(x[base + r * K + col0 + c])));
    }
    const uint32_t byte = scale_byte(block_max(m, s_max));
    const float inverse = scale_inverse(byte);
    for (int64_t i = threadIdx.x; i < rows * kBlock; i += kThreads) {
        const int64_t r = row0 + i / kBlock, c = i % kBlock;
        if (c < cols) {
            const uint8_t q = (uint8_t)pack4(Num<T>::up(x[base + r * K + col0 + c]) * inverse, 0.f, 0.f, 0.f);
            values[base + r * K + col0 + c] = q;
            if (values_t) values_t[base + (col0 + c) * N + r] = q;
        }
    }
    store_block_scales(scales, scales_t, e, n, k, n_blocks, k_blocks, byte);
}

// ---- back -----------------------------------------------------------------------------------------------------------

// A type's largest numbers round up past its range in 8 bits: float16's from 63488 on to 65536, the others' from 248 * 2^120 on to 2^128, which
// fp32 has as an infinity (no value times its scale is one otherwise, and a block with one is NaN). On the way back they are the type's
// largest, so that a gradient made from finite tokens stays finite.
template <typename T>
__device__ __forceinline__ float in_range(float v) {
    if constexpr (std::is_same_v<T, f16_t>) return fabsf(v) == 65536.f ? copysignf(65504.f, v) : v;
    else return fabsf(v) == INFINITY ? copysignf(__uint_as_float(std::is_same_v<T, bf16_t> ? 0x7f7f0000u : 0x7f7fffffu), v) : v;
}

// Eight elements a lane, so that a store of a 16-bit type takes whole lines, four times per workgroup with all loads in front. row_shift: 0, or
// 7 where 128 rows of a matrix of N rows share their scales. Index arithmetic in 32 bits (I32) where the sizes allow it: a 64-bit division costs more than the rest of the kernel.
// [65536, 1408] bf16: 95 -> 53 us (5.2 TB/s). SHIFTED: 2^-shift[row] of every row.
constexpr int kDequantizeUnroll = 4;
template <typename T, bool I32, bool SHIFTED>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* __restrict__ values, const uint8_t* __restrict__ scales,
                                                              const uint8_t* __restrict__ shift, T* __restrict__ out, int64_t total, uint32_t per_row, int64_t K,
                                                              int64_t pitch, int64_t N, int64_t scale_rows, int row_shift) {
    typedef std::conditional_t<I32, uint32_t, int64_t> index;
    const int64_t first = (int64_t)blockIdx.x * (kDequantizeUnroll * kThreads) + threadIdx.x;
    uint2 q[kDequantizeUnroll];
    float scale[kDequantizeUnroll];
    int64_t at[kDequantizeUnroll];
#pragma unroll
    for (int i = 0; i < kDequantizeUnroll; ++i) {
        const int64_t u = first + i * kThreads;
        at[i] = -1;
        if (u < total) {
            const index row = (index)u / (index)per_row, k = ((index)u - row * (index)per_row) * 8;
            index s_row = row;
            if (row_shift) {
                const index e = row / (index)N;
                s_row = e * (index)scale_rows + ((row - e * (index)N) >> row_shift);
            }
            at[i] = (int64_t)row * K + k;
            q[i] = *reinterpret_cast<const uint2*>(values + at[i]);
            scale[i] = scale_value(scales[(int64_t)s_row * pitch + k / kBlock]);
            if constexpr (SHIFTED) scale[i] *= __uint_as_float((127u - shift[row]) << 23);
        }
    }
#pragma unroll
    for (int i = 0; i < kDequantizeUnroll; ++i) {
        if (at[i] < 0) continue;
        const uint32_t w[2] = {q[i].x, q[i].y};
        float f[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float g[4];
            unpack4(w[j], g);
#pragma unroll
            for (int x = 0; x < 4; ++x) f[4 * j + x] = in_range<T>(g[x] * scale[i]);
        }
        if constexpr (sizeof(T) == 4) {
            store_floats(out + at[i], f);
        } else {
            using EL = std::conditional_t<std::is_same_v<T, bf16_t>, ::fmahip::gemm::ElemBf16, ::fmahip::gemm::ElemF16>;
            uint4 v;
            v.x = EL::pack2(f[0], f[1]);
            v.y = EL::pack2(f[2], f[3]);
            v.z = EL::pack2(f[4], f[5]);
            v.w = EL::pack2(f[6], f[7]);
            store_streaming16(reinterpret_cast<uint4*>(out + at[i]), v);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_generic_kernel(const uint8_t* __restrict__ values,
                                                                      const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                                      int64_t total, int64_t K, int64_t pitch, int64_t N,
                                                                      int64_t scale_rows, int row_shift) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
        const int64_t row = i / K, k = i - row * K;
        const int64_t e = row / N, s_row = e * scale_rows + ((row - e * N) >> row_shift);
        float g[4];
        unpack4(values[i], g);
        out[i] = Num<T>::down(in_range<T>(g[0] * scale_value(scales[s_row * pitch + k / kBlock])));
    }
}

template <typename T>
int quantize_rows(const void* x, uint8_t* values, uint8_t* scales, int64_t R, int64_t K, hipStream_t st) {
    const int64_t pitch = scale_pitch(K);
    constexpr int kUnroll = sizeof(T) == 4 ? 1 : 2;
    const int64_t units = R * (pitch / 4), per = (int64_t)kUnroll * (kThreads / 32), grid = (units + per - 1) / per;
    // (2^27 and more short rows take the kernel whose workgroups make several turns)
    const bool vec = K % 16 == 0 && aligned16(x) && aligned16(values) && (reinterpret_cast<uintptr_t>(scales) & 3u) == 0 && grid <= kMostWorkgroups;
    if (vec) {
        hipLaunchKernelGGL((quantize_rows_kernel<T, kUnroll>), dim3((uint32_t)grid), dim3(kThreads), 0, st, (const T*)x, values, (uint32_t*)scales,
                           units, (uint32_t)(pitch / 4), K);
    } else {
        const int64_t total = R * pitch, blocks = (total + kThreads / 8 - 1) / (kThreads / 8);
        const dim3 grid((uint32_t)(blocks < (1 << 16) ? blocks : (1 << 16)));
        hipLaunchKernelGGL(quantize_rows_generic_kernel<T>, grid, dim3(kThreads), 0, st, (const T*)x, values, scales, total, pitch, K);
    }
    return launch_status("quantize_fp8_rows");
}

template <typename T>
int quantize_blocks(const void* x, uint8_t* values, uint8_t* scales, uint8_t* values_t, uint8_t* scales_t, int64_t E, int64_t N, int64_t K,
                    hipStream_t st) {
    const int64_t n_blocks = (N + kBlock - 1) / kBlock, k_blocks = (K + kBlock - 1) / kBlock;
    const dim3 grid((uint32_t)(E * n_blocks * k_blocks));
    const bool vec = K % 8 == 0 && (!values_t || N % 8 == 0) && aligned16(x) && (reinterpret_cast<uintptr_t>(values) & 7u) == 0 &&
                     (reinterpret_cast<uintptr_t>(values_t) & 7u) == 0;
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, (const T*)x, values, scales, values_t, scales_t, N, K, (uint32_t)n_blocks,
                           (uint32_t)k_blocks);
    };
    if (!vec) run(quantize_blocks_generic_kernel<T>);
    else if (values_t) run(quantize_blocks_kernel<T, true>);
    else run(quantize_blocks_kernel<T, false>);
    return launch_status("quantize_fp8_blocks");
}

template <typename T>
int dequantize(const uint8_t* values, const uint8_t* scales, void* out, int64_t E, int64_t N, int64_t K, int64_t block_rows,
               hipStream_t st) {
    const int64_t pitch = scale_pitch(K), scale_rows = (N + block_rows - 1) / block_rows;
    const int shift = block_rows == 1 ? 0 : 7;
    constexpr int64_t per = kDequantizeUnroll * kThreads;
    const int64_t total = E * N * (K / 8), workgroups = (total + per - 1) / per;
    if (K % 8 == 0 && (reinterpret_cast<uintptr_t>(values) & 7u) == 0 && aligned16(out) && workgroups <= kMostWorkgroups) {
        const dim3 grid((uint32_t)workgroups);
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, values, scales, nullptr, (T*)out, total, (uint32_t)(K / 8), K, pitch, N, scale_rows,
                               shift);
        };
        if (total + per < (1ll << 31)) run(dequantize_kernel<T, true, false>);
        else run(dequantize_kernel<T, false, false>);
    } else {
        const int64_t elements = E * N * K, blocks = (elements + kThreads - 1) / kThreads;
        const dim3 grid((uint32_t)(blocks < (1 << 20) ? blocks : (1 << 20)));
        hipLaunchKernelGGL(dequantize_generic_kernel<T>, grid, dim3(kThreads), 0, st, values, scales, (T*)out, elements, K, pitch, N, scale_rows,
                           shift);
    }
    return launch_status("dequantize_fp8");
}

int check_matrix(const char* who, int64_t E, int64_t N, int64_t K, int64_t block_rows, int dtype) {
    FMA_REQUIRE(dtype_bytes(dtype) != 0, FMA_ERR_BAD_DTYPE, "%s: dtype code %d", who, dtype);
    FMA_REQUIRE(E >= 0 && N >= 0 && K >= 1, FMA_ERR_BAD_SIZE, "%s: bad size E=%lld N=%lld K=%lld", who, (long long)E, (long long)N, (long long)K);
    FMA_REQUIRE(block_rows == 1 || block_rows == kBlock, FMA_ERR_BAD_SIZE, "%s: blocks have 1 or 128 rows, not %lld", who, (long long)block_rows);
    // (64-bit offsets in the kernels; what is limited is K / 16 and the number of units of 512 elements)
    FMA_REQUIRE(K <= (1ll << 31) && N <= (1ll << 40) && E <= (1ll << 31), FMA_ERR_TOO_MANY_ELEMENTS, "%s: K <= 2^31", who);
    const int64_t units = block_rows == 1 ? (K + 511) / 512 : (K + 127) / 128;
    const int64_t rows = block_rows == 1 ? N : (N + 127) / 128;
    FMA_REQUIRE(E == 0 || rows == 0 || units * rows <= ((1ll << 31) - 1) / E, FMA_ERR_TOO_MANY_ELEMENTS,
                "%s: more than 2^31 - 1 pieces of 512 elements of a row, or blocks of 128 x 128", who);
    return FMA_OK;
}

}  // namespace

int fp8::dequantize_shifted(const uint8_t* values, const uint8_t* scales, const uint8_t* shift, void* out, int64_t R, int64_t K, hipStream_t st) {
    const int64_t total = R * (K / 8), per = kDequantizeUnroll * kThreads;
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((uint32_t)((total + per - 1) / per)), dim3(kThreads), 0, st, values, scales, shift, (f16_t*)out, total,
                           (uint32_t)(K / 8), K, scale_pitch(K), R, R, 0);
    };
    if (total + per < (1ll << 31)) run(dequantize_kernel<f16_t, true, true>);
    else run(dequantize_kernel<f16_t, false, true>);
    return launch_status("dequantize_fp8");
}

}  // namespace fmahip

extern "C" {

int64_t fma_fp8_scale_pitch(int64_t K) { return K > 0 ? fmahip::fp8::scale_pitch(K) : 0; }

int fma_quantize_fp8(const void* x, void* values, void* scales, void* values_t, void* scales_t, int64_t E, int64_t N, int64_t K,
                     int64_t block_rows, int dtype, void* stream) {
    using namespace fmahip;
    if (const int rc = check_matrix("quantize_fp8", E, N, K, block_rows, dtype)) return rc;
    FMA_REQUIRE(!values_t == !scales_t, FMA_ERR_NULL_POINTER, "quantize_fp8: the transposed copy takes values and scales");
    FMA_REQUIRE(!values_t || block_rows == 128, FMA_ERR_UNSUPPORTED, "quantize_fp8: a transposed copy exists of 128 x 128 blocks only");
    if (E == 0 || N == 0) return FMA_OK;
    FMA_REQUIRE(block_rows == 1 || E * ((N + 127) / 128) * ((K + 127) / 128) <= kMostWorkgroups, FMA_ERR_TOO_MANY_ELEMENTS,
                "quantize_fp8: more than 2^24 - 1 blocks of 128 x 128");
    FMA_REQUIRE(x && values && scales, FMA_ERR_NULL_POINTER, "quantize_fp8: x, values or scales is NULL");
    FMA_REQUIRE((reinterpret_cast<uintptr_t>(x) & (uintptr_t)(dtype_bytes(dtype) - 1)) == 0, FMA_ERR_MISALIGNED, "quantize_fp8: x is not aligned to its elements");
    hipStream_t st = (hipStream_t)stream;
    uint8_t *v = (uint8_t*)values, *s = (uint8_t*)scales, *vt = (uint8_t*)values_t, *t = (uint8_t*)scales_t;
    if (block_rows == 1) {
        if (dtype == FMA_F32) return quantize_rows<float>(x, v, s, E * N, K, st);
        if (dtype == FMA_F16) return quantize_rows<f16_t>(x, v, s, E * N, K, st);
        return quantize_rows<bf16_t>(x, v, s, E * N, K, st);
    }
    if (dtype == FMA_F32) return quantize_blocks<float>(x, v, s, vt, t, E, N, K, st);
    if (dtype == FMA_F16) return quantize_blocks<f16_t>(x, v, s, vt, t, E, N, K, st);
    return quantize_blocks<bf16_t>(x, v, s, vt, t, E, N, K, st);
}

int fma_dequantize_fp8(const void* values, const void* scales, void* out, int64_t E, int64_t N, int64_t K, int64_t block_rows, int dtype,
                       void* stream) {
    using namespace fmahip;
    if (const int rc = check_matrix("dequantize_fp8", E, N, K, block_rows, dtype)) return rc;
    if (E == 0 || N == 0) return FMA_OK;
    FMA_REQUIRE(values && scales && out, FMA_ERR_NULL_POINTER, "dequantize_fp8: values, scales or out is NULL");
    FMA_REQUIRE((reinterpret_cast<uintptr_t>(out) & (uintptr_t)(dtype_bytes(dtype) - 1)) == 0, FMA_ERR_MISALIGNED, "dequantize_fp8: out is not aligned to its elements");
    hipStream_t st = (hipStream_t)stream;
    const uint8_t *v = (const uint8_t*)values, *s = (const uint8_t*)scales;
    if (dtype == FMA_F32) return dequantize<float>(v, s, out, E, N, K, block_rows, st);
    if (dtype == FMA_F16) return dequantize<f16_t>(v, s, out, E, N, K, block_rows, st);
    return dequantize<bf16_t>(v, s, out, E, N, K, block_rows, st);
}

}  // extern "C"
