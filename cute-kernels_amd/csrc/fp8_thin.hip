// Products of 8-bit weights with a few rows per group (a decode step). What bounds them is the stream of the weights, one byte per element
// against a handful of rows.
//
// The unit of work is 32 weight rows of one expert (16 of "up" and 16 of "gate" with the activation) against up to 16 or 32 rows, the
// reduction in KS parts, one wavefront each, whose sums are added up through LDS in a fixed order. Weights go straight to registers, 16 bytes a lane, as
// the matrix instruction takes them (16 rows x 64 bytes a load, two loads a line). Without the non-temporal hint: the line is asked for
// twice, and with it the halves come from memory one by one (128 x 4 rows, 4096 x 1536, 174 -> 140 us without; 8 x 4, 4096 x 14336, 98 -> 83).
// Many small wavefronts keep the loads in flight; there is no barrier in the loop. (Rows in LDS for eight units at a time, with a barrier
// per 512 elements: 8 x 4 rows, 28672 x 4096, 212 us against 168.)
//
// The rows come from memory in 8 bits (the product of quantised operands), or are quantised on the way to the instruction: the tokens of a
// layer (16 bits) and the activation between its two products (fp32). Each lane has 32 elements of a block of 128, its three neighbours
// the rest; every wavefront of an expert quantises the same rows anew, 120 vector instructions per 4 KB of weights, which costs less than a
// launch that does it once. The first product, whose sums become e4m3 activations, is one of bfloat16 instructions (the 8-bit one cuts
// products at 2^-13 of the largest of eight: one activation in 2000 was rounded to the other side of a border, a token off by 0.004 instead of
// 0.0016): 48 conversions and 6 matrix instructions more per 4 KB, 0 to 5 % of a step of 1 to 64 tokens (hidden 2048, I 1408, E 64, k 8, us:
// 29.6, 64, 112.5, 163.3 -> 30.1, 66, 115.5, 165.1 at 1, 4, 16 and 64; 4096 x 14336, E 8, k 2: 87.8, 194, 289, 446 -> 91.3, 197, 288, 448).
// An expert's rows are found by looking through the ids, so that a decode step needs no routing index.
#include "fp8_thin.h"
#include "gemm_parts.h"

namespace fmahip {
namespace fp8 {
namespace {

using ::fmahip::gemm::bf16x2;
using ::fmahip::gemm::bf16x8;
using ::fmahip::gemm::kOutOfRange;
using ::fmahip::gemm::uniform;

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;

enum Rows { ROWS_FP8, ROWS_BF16, ROWS_F16, ROWS_F32 };
enum Out { OUT_BF16, OUT_F16, OUT_F32, OUT_GLU };

struct ThinArgs {
    const uint8_t *W, *W_s;
    const void* x;           // rows
    const uint8_t* x_s;      // ROWS_FP8: their scales
    const uint32_t* sizes;   // ROWS_FP8: rows per group, one behind the other; NULL: one group of R
    const void* ids;         // otherwise: the expert of every slot
    int id_bytes;
    uint32_t divisor;        // slot / divisor is the row of x
    uint32_t E, R, N, K, x_rows;
    uint32_t s_pitch;        // scales of K elements
    void* out;               // [R, N]
    uint32_t col_blocks;     // units per group
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0);
}

// 32 e4m3 values and their scale (the low byte) as bfloat16, which holds the products exactly
__device__ __forceinline__ void widen(bf16x8 (&to)[4], i32x8 raw, uint32_t scale) {
    const float factor = __uint_as_float((scale & 255u) << 23);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
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
}

// One unit: rows `first` .. of the group's list (`rows` of them, at most 16 * TB).
template <int SRC, int OUT, int TB, int KS>
struct Unit {
    static constexpr int kUnroll = SRC == ROWS_FP8 ? 4 : 2;
    static constexpr int kElem = SRC == ROWS_FP8 ? 1 : (SRC == ROWS_F32 ? 4 : 2);  // bytes
    static constexpr int kVec = 2 * kElem;                                         // 16-byte loads of 32 elements

    static __device__ __forceinline__ void run(const ThinArgs& a, uint32_t e, uint32_t n0, const uint32_t* list, uint32_t rows, float* parts) {
        constexpr bool kGlu = OUT == OUT_GLU;
        const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6);
        const uint32_t r16 = lane & 15u, q = lane >> 4;
        const uint32_t K = a.K, N = a.N;
        const uint32_t k_blocks = (K + kBlock - 1) / kBlock;
        // this wavefront's blocks of the reduction
        const uint32_t per = (k_blocks + KS - 1) / KS, k0 = wave * per, k1 = k0 + per < k_blocks ? k0 + per : k_blocks;

        // weights: fragment 0 and 1; rows past the last one are out of range
        const uint64_t matrix = (uint64_t)N * K;
        const uint8_t* const base = a.W + (kGlu ? 2 : 1) * e * matrix + (uint64_t)n0 * K;
        const uint32_t bytes = (N - n0 < 32u ? N - n0 : 32u) * K;
        const __amdgpu_buffer_rsrc_t w0 = buffer(base, bytes), w1 = buffer(kGlu ? base + matrix : base, bytes);
        uint32_t w_off[2];
        if constexpr (kGlu) {
            w_off[0] = w_off[1] = r16 * K + q * 16u;
        } else {  // rows 8 a + b, and 8 a + 4 + b: a lane's results are eight neighbouring columns
            w_off[0] = ((r16 >> 2) * 8u + (r16 & 3u)) * K + q * 16u;
            w_off[1] = w_off[0] + 4u * K;
        }
        const uint32_t n_blocks = (N + kBlock - 1) / kBlock;
        typedef const __attribute__((address_space(4))) uint32_t* const_words;  // read by scalar loads
        const uint8_t* const s_base = a.W_s + ((uint64_t)(kGlu ? 2 : 1) * e * n_blocks + n0 / kBlock) * a.s_pitch;
        const const_words ws0 = (const_words)s_base, ws1 = (const_words)(s_base + (kGlu ? (uint64_t)n_blocks * a.s_pitch : 0));

        // rows
        const __amdgpu_buffer_rsrc_t xr = buffer(a.x, a.x_rows * K * (uint32_t)kElem);
        const __amdgpu_buffer_rsrc_t xs = buffer(a.x_s, SRC == ROWS_FP8 ? a.x_rows * a.s_pitch : 0u);
        uint32_t x_off[TB], s_off[TB];
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const uint32_t r = (uint32_t)t * 16u + r16;
            const uint32_t src = r < rows ? list[r] / a.divisor : a.x_rows;
            x_off[t] = src < a.x_rows ? src * K * (uint32_t)kElem + q * 16u * (uint32_t)kElem : kOutOfRange;
            s_off[t] = src < a.x_rows ? src * a.s_pitch : kOutOfRange;
        }

        f32x4 acc[TB][2];
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[t][0] = acc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};

        for (uint32_t kb = k0; kb < k1; kb += kUnroll) {
            u32x4 wl[kUnroll][2][2], xl[kUnroll][TB][2 * kElem];
            uint32_t wsc[kUnroll][2], xsc[kUnroll][TB];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const uint32_t k = kb + (uint32_t)u;
                const bool on = k < k1;  // a step past the last one multiplies zeros
                const bool lo = on && k * kBlock + q * 16u < K, hi = on && k * kBlock + 64u + q * 16u < K;
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    wl[u][f][0] = load16(f ? w1 : w0, lo ? w_off[f] + k * kBlock : kOutOfRange);
                    wl[u][f][1] = load16(f ? w1 : w0, hi ? w_off[f] + k * kBlock + 64u : kOutOfRange);
                }
                const uint32_t word = on ? k >> 2 : 0u, shift = (k & 3u) * 8u;
                wsc[u][0] = on ? ws0[word] >> shift : 127u;
                wsc[u][1] = kGlu ? (on ? ws1[word] >> shift : 127u) : wsc[u][0];
#pragma unroll
                for (int t = 0; t < TB; ++t) {
#pragma unroll
                    for (int i = 0; i < 2 * kElem; ++i) {
                        const bool in = i < kElem ? lo : hi;
                        const uint32_t at = x_off[t] + (k * kBlock + (i < kElem ? 0u : 64u)) * (uint32_t)kElem + (uint32_t)(i % kElem) * 16u;
                        xl[u][t][i] = load16(xr, in && x_off[t] != kOutOfRange ? at : kOutOfRange);
                    }
                    if constexpr (SRC == ROWS_FP8)
                        xsc[u][t] = __builtin_amdgcn_raw_buffer_load_b32(xs, (int)(on && s_off[t] != kOutOfRange ? s_off[t] + word * 4u : kOutOfRange), 0, 0) >> shift;
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const bool on = kb + (uint32_t)u < k1;
                i32x8 w[2];
                bf16x8 ww[2][4];
#pragma unroll
                for (int f = 0; f < 2; ++f) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[f][i] = (int)wl[u][f][i / 4][i % 4];
                    if constexpr (kGlu) widen(ww[f], w[f], wsc[u][f]);
                }
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    i32x8 x;
                    uint32_t byte;
                    if constexpr (SRC == ROWS_FP8) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = (int)xl[u][t][i / 4][i % 4];
                        byte = on ? xsc[u][t] : 127u;
                    } else {
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const uint32_t word = xl[u][t][i * kElem / 16][i * kElem / 4 % 4];
                            if constexpr (SRC == ROWS_F32) v[i] = __uint_as_float(word);
                            else if constexpr (SRC == ROWS_BF16) v[i] = i % 2 ? __uint_as_float(word & 0xffff0000u) : bf16_bits_to_float(word);
                            else v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(word >> (i % 2 * 16)));
                        }
                        uint32_t m = 0;
#pragma unroll
                        for (int i = 0; i < 32; ++i) m = max_u32(m, magnitude_bits(v[i]));
                        m = max_u32(m, (uint32_t)__shfl_xor((int)m, 16, 64));
                        m = max_u32(m, (uint32_t)__shfl_xor((int)m, 32, 64));
                        byte = scale_byte(m);
                        const float inverse = scale_inverse(byte);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            x[i] = (int)pack4(v[4 * i] * inverse, v[4 * i + 1] * inverse, v[4 * i + 2] * inverse, v[4 * i + 3] * inverse);
                    }
                    if constexpr (kGlu) {
                        bf16x8 xw[4];
                        widen(xw, x, byte);
#pragma unroll
                        for (int s = 0; s < 4; ++s)
#pragma unroll
                            for (int f = 0; f < 2; ++f) acc[t][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[f][s], xw[s], acc[t][f], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int f = 0; f < 2; ++f)
                            acc[t][f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[f], x, acc[t][f], 0, 0, 0, (int)wsc[u][f], 0, (int)byte);
                    }
                }
            }
        }

        // ---- sums of the parts, in their order ----
        if constexpr (KS > 1) {
            __syncthreads();  // (the parts of the pass before have been read)
            if (wave) {
#pragma unroll
                for (int t = 0; t < TB; ++t)
#pragma unroll
                    for (int f = 0; f < 2; ++f) *reinterpret_cast<f32x4*>(parts + ((((wave - 1u) * TB + t) * 2 + f) * 64 + lane) * 4) = acc[t][f];
            }
            __syncthreads();
            if (wave) return;
            for (int s = 0; s < KS - 1; ++s)
#pragma unroll
                for (int t = 0; t < TB; ++t)
#pragma unroll
                    for (int f = 0; f < 2; ++f) acc[t][f] += *reinterpret_cast<const f32x4*>(parts + (((s * TB + t) * 2 + f) * 64 + lane) * 4);
        }
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const uint32_t r = (uint32_t)t * 16u + r16;
            if (r >= rows) continue;
            const uint64_t row = list[r];
            if constexpr (kGlu) {
                f32x4 y;
#pragma unroll
                for (int x = 0; x < 4; ++x) y[x] = acc[t][0][x] * acc[t][1][x] * sigmoid_clamped_fast(acc[t][1][x]);
                if (n0 + q * 4u < N) *reinterpret_cast<f32x4*>((float*)a.out + row * N + n0 + q * 4u) = y;
            } else {
                using T = std::conditional_t<OUT == OUT_BF16, bf16_t, std::conditional_t<OUT == OUT_F16, f16_t, float>>;
                const uint32_t col = n0 + q * 8u;
                T* const to = (T*)a.out + row * N + col;
                if (N % 8u == 0) {
                    if (col < N) {
                        constexpr int V = Vec16<T>::N;
#pragma unroll
                        for (int c = 0; c < 8 / V; ++c) {
                            Vec16<T> v;
#pragma unroll
                            for (int x = 0; x < V; ++x) v.v[x] = Num<T>::down(acc[t][(c * V + x) / 4][(c * V + x) % 4]);
                            *(reinterpret_cast<Vec16<T>*>(to) + c) = v;
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        if (col + x < N) to[x] = Num<T>::down(acc[t][x / 4][x % 4]);
                }
            }
        }
    }
};

// Workgroup = KS wavefronts: one unit of one group, all passes of 16 * TB of its rows one after the other.
template <int SRC, int OUT, int TB, int KS>
__global__ __launch_bounds__(64 * KS) void fp8_thin_kernel(const ThinArgs a) {
    constexpr uint32_t kPass = 16 * TB;
    constexpr uint32_t kList = SRC == ROWS_FP8 ? kPass : (uint32_t)kMaxThinSlots;
    __shared__ uint32_t s_list[kList];
    __shared__ __attribute__((aligned(16))) float s_parts[KS > 1 ? (KS - 1) * TB * 2 * 64 * 4 : 4];
    __shared__ uint32_t s_count;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t e = blockIdx.x / a.col_blocks;
    const uint32_t n0 = (blockIdx.x - e * a.col_blocks) * (OUT == OUT_GLU ? 16u : 32u);
    uint32_t rows, first = 0;
    if constexpr (SRC == ROWS_FP8) {
        if (a.sizes) {  // rows past R do not exist, whatever the sizes say
            uint64_t before = 0;
            for (uint32_t base = 0; base < e; base += 64) before += base + lane < e ? a.sizes[base + lane] : 0u;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d, 64);
            first = before < a.R ? (uint32_t)before : a.R;
            const uint32_t m = a.sizes[e];
            rows = m < a.R - first ? m : a.R - first;
        } else {
            rows = a.R;
        }
    } else {
        // `e` counts the experts that have a slot: which one it is, from a bit for each of them
        constexpr uint32_t kWords = FMA_MAX_GROUPS / 32;
        __shared__ uint32_t s_named[kWords];
        if (threadIdx.x < 64) {
            if (lane < kWords) s_named[lane] = 0u;
            for (uint32_t s = lane; s < a.R; s += 64) {
                const int64_t id = a.id_bytes == 8 ? ((const int64_t*)a.ids)[s] : (int64_t)((const int32_t*)a.ids)[s];
                if ((uint64_t)id < a.E) atomicOr(&s_named[(uint32_t)id >> 5], 1u << ((uint32_t)id & 31u));
            }
            const uint32_t word = lane < kWords ? s_named[lane] : 0u;
            const uint32_t n = (uint32_t)__popc(word), before = wave_inclusive_scan<uint32_t>(n) - n;
            const uint64_t mine = __ballot(before <= e && e < before + n);
            uint32_t found = a.E;
            if (mine) {
                const int src = (int)__builtin_ctzll(mine);
                uint32_t bits = (uint32_t)__shfl((int)word, src, 64);
                for (uint32_t skip = e - (uint32_t)__shfl((int)before, src, 64); skip; --skip) bits &= bits - 1u;
                found = (uint32_t)src * 32u + (uint32_t)__builtin_ctz(bits);
            }
            if (lane == 0) s_count = found;
        }
        __syncthreads();
        e = s_count;
        if (e >= a.E) return;
        __syncthreads();
        // its slots, in their order
        if (threadIdx.x < 64) {
            uint32_t n = 0;
            for (uint32_t base = 0; base < a.R; base += 64) {
                const uint32_t s = base + lane;
                int64_t id = -1;
                if (s < a.R) id = a.id_bytes == 8 ? ((const int64_t*)a.ids)[s] : (int64_t)((const int32_t*)a.ids)[s];
                const uint64_t mask = __ballot(id == (int64_t)e);
                if (id == (int64_t)e) s_list[n + (uint32_t)__popcll(mask & ((1ull << lane) - 1ull))] = s;
                n += (uint32_t)__popcll(mask);
            }
            if (lane == 0) s_count = n;
        }
        __syncthreads();
        rows = s_count;
    }
    rows = uniform(rows);
    first = uniform(first);
    for (uint32_t at = 0; at < rows; at += kPass) {
        const uint32_t here = rows - at < kPass ? rows - at : kPass;
        const uint32_t* list = s_list + at;
        if constexpr (SRC == ROWS_FP8) {
            __syncthreads();
            if (threadIdx.x < here) s_list[threadIdx.x] = first + at + threadIdx.x;
            __syncthreads();
            list = s_list;
        }
        if (TB > 1 && here <= 16u) Unit<SRC, OUT, 1, KS>::run(a, e, n0, list, here, s_parts);
        else Unit<SRC, OUT, TB, KS>::run(a, e, n0, list, here, s_parts);
    }
}

template <int SRC, int OUT>
int launch(const char* who, ThinArgs a, hipStream_t st) {
    const uint32_t per = OUT == OUT_GLU ? 16u : 32u;
    a.col_blocks = (a.N + per - 1) / per;
    const int64_t groups = a.E < a.R ? a.E : a.R, cus = num_compute_units() > 0 ? num_compute_units() : 256;
    // Passes of 32 rows where groups of more than 16, which passes of 16 stream their weights twice for, are to be expected: their 25 registers more
    // cost otherwise. 16 / 32, us, at 4, 8, 10, 16 rows a group on average: 8 x 4096 x 14336 83, 88, 105, 130 / 92, 95, 101, 111; 8 x 2048 x
    // 8192 31, 32, 41, 54 / 34, 35, 36, 40; 8 x 28672 x 4096 163, 167, 187, 237 / 161, 165, 174, 202; 64 x 2816 x 2048 64, 69, 73, 101 / 64, 67, 71, 83.
    const bool wide = (int64_t)a.R > 8 * groups;
    // parts of the reduction, of two blocks at least, until there are 32 wavefronts per compute unit, two rounds (12: 8 x 4 rows, 28672 x 4096,
    // 179 -> 169 us; 64: 64 x 16 rows, 2816 x 2048, 84 -> 96)
    const int64_t units = groups * a.col_blocks, k_blocks = (a.K + kBlock - 1) / kBlock;
    int parts = 1;
    while (parts < 8 && units * parts < 32 * cus && k_blocks >= 4 * parts) parts *= 2;
    const dim3 grid((uint32_t)(SRC == ROWS_FP8 ? a.E : groups) * a.col_blocks);
    auto run = [&](auto kernel, int ks) { hipLaunchKernelGGL(kernel, grid, dim3(64 * ks), 0, st, a); };
    if (wide) {
        if (parts == 1) run(fp8_thin_kernel<SRC, OUT, 2, 1>, 1);
        else if (parts == 2) run(fp8_thin_kernel<SRC, OUT, 2, 2>, 2);
        else if (parts == 4) run(fp8_thin_kernel<SRC, OUT, 2, 4>, 4);
        else run(fp8_thin_kernel<SRC, OUT, 2, 8>, 8);
    } else {
        if (parts == 1) run(fp8_thin_kernel<SRC, OUT, 1, 1>, 1);
        else if (parts == 2) run(fp8_thin_kernel<SRC, OUT, 1, 2>, 2);
        else if (parts == 4) run(fp8_thin_kernel<SRC, OUT, 1, 4>, 4);
        else run(fp8_thin_kernel<SRC, OUT, 1, 8>, 8);
    }
    return launch_status(who);
}

}  // namespace

namespace {
// Whether this kernel is ahead of the tiles, of which a round takes 1.75 us a block of the reduction, one of a few tiles 1.3. Here the weights
// stream at 5.4 TB/s, less an eightieth per row of the average group, and twice as long from 16 rows on. Weights from memory, this / tiles, us,
// at 4, 8, 16 and 32 rows: 8 x 28672 x 4096 169, 171, 204, 325 / 232; 128 x 4096 x 1536 140, 157, 180, 256 / 160; 64 x 2816 x 2048 66, 70, 84, 127
// / 81; 32 x 5760 x 2880 101, 111, 128, 174 / 110; 64 x 2048 x 1408 40, 42, 49, 76 / 42; 8 x 4096 x 14336 84, 89, 112, 192 / 144; 8 x 2048 x 8192
// 33, 34, 41, 70 / 85.
bool few_rows(int64_t E, int64_t R, int64_t N, int64_t K) {
    const int64_t groups = E < R ? E : R, cus = num_compute_units() > 0 ? num_compute_units() : 256;
    if (R > 32 * groups) return false;
    const int64_t tiles = groups * ((N + 255) / 256), rounds = (tiles + cus - 1) / cus;
    const double row = (double)R / groups, stream = (double)groups * N * K * (row > 16 ? 1.9 : 1 + row / 80) / 5.4e6;
    return stream <= 3 + (double)rounds * ((K + kBlock - 1) / kBlock) * (tiles <= cus ? 1.3 : 1.75);
}
// lane offsets into the rows, and the number of threads of a launch
bool fits(int64_t E, int64_t R, int64_t N, int64_t K, int64_t bytes, int64_t per) {
    return R * K * bytes < (1ll << 31) && E * ((N + per - 1) / per) < (1ll << 22);
}
}  // namespace

bool is_thin_product(int64_t E, int64_t R, int64_t N, int64_t K) { return fits(E, R, N, K, 1, 32) && few_rows(E, R, N, K); }
bool are_thin_experts(int64_t E, int64_t R, int64_t H, int64_t I) {
    return R <= kMaxThinSlots && fits(E, R, I, H, 2, 16) && fits(E, R, H, I, 4, 32) && few_rows(E, R, 2 * I, H);
}

int launch_thin_product(const void* A, const void* A_s, const void* B, const void* B_s, void* D, const uint32_t* sizes, int64_t E, int64_t R,
                        int64_t N, int64_t K, int dtype, hipStream_t st) {
    ThinArgs a = {};
    a.W = (const uint8_t*)B;
    a.W_s = (const uint8_t*)B_s;
    a.x = A;
    a.x_s = (const uint8_t*)A_s;
    a.sizes = sizes;
    a.divisor = 1;
    a.E = (uint32_t)E;
    a.R = a.x_rows = (uint32_t)R;
    a.N = (uint32_t)N;
    a.K = (uint32_t)K;
    a.s_pitch = (uint32_t)scale_pitch(K);
    a.out = D;
    if (dtype == FMA_F32) return launch<ROWS_FP8, OUT_F32>("grouped_gemm_fp8", a, st);
    if (dtype == FMA_F16) return launch<ROWS_FP8, OUT_F16>("grouped_gemm_fp8", a, st);
    return launch<ROWS_FP8, OUT_BF16>("grouped_gemm_fp8", a, st);
}

int launch_thin_experts(const void* x, const void* ids, int id_bytes, const void* W1, const void* W1_s, const void* W2, const void* W2_s, float* act,
                        float* o, int64_t T, int64_t top_k, int64_t E, int64_t H, int64_t I, int dtype, hipStream_t st) {
    ThinArgs a = {};
    a.W = (const uint8_t*)W1;
    a.W_s = (const uint8_t*)W1_s;
    a.x = x;
    a.ids = ids;
    a.id_bytes = id_bytes;
    a.divisor = (uint32_t)top_k;
    a.E = (uint32_t)E;
    a.R = (uint32_t)(T * top_k);
    a.x_rows = (uint32_t)T;
    a.N = (uint32_t)I;
    a.K = (uint32_t)H;
    a.s_pitch = (uint32_t)scale_pitch(H);
    a.out = act;
    const int rc = dtype == FMA_BF16 ? launch<ROWS_BF16, OUT_GLU>("swiglu_experts_fp8", a, st) : launch<ROWS_F16, OUT_GLU>("swiglu_experts_fp8", a, st);
    if (rc) return rc;
    a.W = (const uint8_t*)W2;
    a.W_s = (const uint8_t*)W2_s;
    a.x = act;
    a.divisor = 1;
    a.x_rows = a.R;
    a.N = (uint32_t)H;
    a.K = (uint32_t)I;
    a.s_pitch = (uint32_t)scale_pitch(I);
    a.out = o;
    return launch<ROWS_F32, OUT_F32>("swiglu_experts_fp8", a, st);
}

}  // namespace fp8
}  // namespace fmahip
