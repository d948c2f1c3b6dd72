// The experts of a SwiGLU layer in 8 bits, from the tokens to the gated sum, one call per direction:
//
//   forward   x8 = q(x); h_e = x8 W1_e^T; a8 = q(swiglu(h)); o_e = a8 W2_e^T; y[t] = sum_j gates[t, j] o[row of (t, j)]
//   backward  do = gates dy, do8 = q(do); da = do8 W2_e; dh = swiglu'(h8) da, dh8 = q(dh); dx[t] = sum_j (dh8 W1_e)[row of (t, j)];
//             dW2_e = do_e^T a8_e; dW1_e = dh_e^T x8[rows of e]; dgates[t, j] = <dy[t], o[row of (t, j)]>
//
// with q the block format of fp8_parts.h. The tokens are quantised once and gathered inside the first product, the activation is quantised
// in that product's epilogue. What a training step keeps is in 8 bits (tokens, pre-activation, activation; the experts' output, which the
// gates' gradient reads, in 16). The weight gradients are products in 16 bits: of the unrounded gradients' 16-bit form and the 8-bit
// activations, which are exact in bf16 (in fp16 as far as its exponents reach; a row past its range shares a power of two with its gradient).
#include "fp8_gemm_launch.h"
#include "fp8_thin.h"

namespace fmahip {
namespace {
using namespace fp8;

constexpr int kThreads = 256;
constexpr uint32_t kFloat16Scale = 127 + 7;  // 448 * 2^7 = 57344: the largest scale of a block that float16 holds

// Whether a slot's id names an expert: a choice that names none has no row, and takes no part in anything.
__device__ __forceinline__ bool names_expert(const void* ids, int id_bytes, int64_t slot, uint32_t E) {
    const int64_t id = id_bytes == 8 ? ((const int64_t*)ids)[slot] : (int64_t)((const int32_t*)ids)[slot];
    return (uint64_t)id < E;
}

// ---- y[t] = sum_j gates[t, j] * o[inv[t, j]], fp32 sums in ascending j; gates NULL: ones ------------------------------
// o in type O; not INDEXED: the row of a slot is the slot. One workgroup per token and kThreads * 8 columns (64 * 8 of few tokens); KC choices (top_k, or 4 at a time) of a vector are loaded before the first is added.
template <typename T, typename O, bool INDEXED, int KC>
__global__ __launch_bounds__(kThreads) void sum_choices_kernel(const O* __restrict__ o, const void* __restrict__ ids, int id_bytes,
                                                               const int32_t* __restrict__ inv, const T* __restrict__ gates, uint32_t top_k,
                                                               uint32_t E, uint32_t H, int64_t slots, T* __restrict__ y) {
    const int64_t t = blockIdx.x;
    const uint32_t h = (blockIdx.y * blockDim.x + threadIdx.x) * 8u;
    if (h < H) {
        float sum[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.f;
        for (uint32_t j0 = 0; j0 < top_k; j0 += KC) {
            constexpr int V = Vec16<O>::N;
            Vec16<O> v[KC][8 / V];
            float g[KC];
            bool in[KC];
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                // (loads first, looks after: a row that does not count is row 0, and what it holds is dropped)
                const int64_t slot = t * top_k + (j0 + j < top_k ? j0 + j : 0);
                const bool named = j0 + j < top_k && names_expert(ids, id_bytes, slot, E);
                int64_t row = slot;
                if constexpr (INDEXED) row = inv[slot];
                in[j] = named && (uint64_t)row < (uint64_t)slots;
                if (INDEXED && !in[j]) row = 0;
#pragma unroll
                for (int c = 0; c < 8 / V; ++c) v[j][c] = load_streaming16(reinterpret_cast<const Vec16<O>*>(o + row * H + h) + c);
                g[j] = gates ? Num<T>::up(gates[slot]) : 1.0f;
            }
#pragma unroll
            for (int j = 0; j < KC; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] = in[j] ? fmaf(g[j], Num<O>::up(v[j][i / V].v[i % V]), sum[i]) : sum[i];
        }
        Vec16<T> w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w.v[i] = Num<T>::down(sum[i]);
        *reinterpret_cast<Vec16<T>*>(y + t * H + h) = w;
    }
}

// O = T: rows in the routing order, inv; O = float: rows by slot
template <typename T, typename O = T>
int sum_choices(const void* o, const void* ids, int id_bytes, const int32_t* inv, const void* gates, int64_t T_, int64_t top_k, int64_t E,
                int64_t H, void* y, hipStream_t st) {
    const uint32_t threads = T_ < 64 ? 64 : kThreads;
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((uint32_t)T_, (uint32_t)((H + threads * 8 - 1) / (threads * 8))), dim3(threads), 0, st, (const O*)o, ids, id_bytes,
                           inv, (const T*)gates, (uint32_t)top_k, (uint32_t)E, (uint32_t)H, T_ * top_k, (T*)y);
    };
    constexpr bool kIndexed = std::is_same_v<T, O>;
    if (top_k == 1) run(sum_choices_kernel<T, O, kIndexed, 1>);
    else if (top_k == 2) run(sum_choices_kernel<T, O, kIndexed, 2>);
    else if (top_k <= 4 || top_k % 8 != 0) run(sum_choices_kernel<T, O, kIndexed, 4>);
    else run(sum_choices_kernel<T, O, kIndexed, 8>);
    return launch_status("swiglu_experts_fp8");
}

// ---- the combine's backward, and the rows' gradient in 8 bits beside it ----------------------------------------------
// One wavefront per (token, choice): do = gate * dy rounded to T and, from the unrounded products, in 8 bits; dgate = <dy, o>. H % 8 == 0.
//
// SHIFTED (float16): an activation may be past float16's range (its sums are fp32), and the product do^T a8 takes a 16-bit copy of it. A row whose
// largest block has a scale of 2^(7 + s), s > 0, gives that copy 2^-s of its activations, 57344 at most, and do 2^s of its gradient, which leaves every
// product what it is: powers of two, written to `shift`. (A do that overflows by that belongs to a product of 2^30 and more.)
template <typename T, bool SHIFTED>
__global__ __launch_bounds__(kThreads) void combine_bwd_fp8_kernel(const T* __restrict__ dy, const T* __restrict__ o,
                                                                   const void* __restrict__ ids, int id_bytes,
                                                                   const int32_t* __restrict__ inv, const T* __restrict__ gates,
                                                                   int64_t slots, uint32_t top_k, uint32_t E, uint32_t H, T* __restrict__ d_o,
                                                                   uint8_t* __restrict__ values, uint32_t* __restrict__ scales,
                                                                   T* __restrict__ d_gates, const uint8_t* __restrict__ a8_s, uint32_t a_blocks,
                                                               uint32_t a_pitch, uint8_t* __restrict__ shift) {
    const uint32_t lane = threadIdx.x & 63u;
    const int64_t slot = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 64;
    if (slot >= slots) return;
    const int64_t row = names_expert(ids, id_bytes, slot, E) ? inv[slot] : -1;
    if ((uint64_t)row >= (uint64_t)slots) {
        if (d_gates && lane == 0) d_gates[slot] = Num<T>::down(0.f);
        return;
    }
    const float gate = Num<T>::up(gates[slot]);
    const uint32_t quads = (H + 511u) / 512u;
    float raise = 1.f;
    if constexpr (SHIFTED) {
        uint32_t top = 0;
        for (uint32_t b = lane; b < a_blocks; b += 64u) {
            const uint32_t byte = a8_s[row * a_pitch + b];
            top = max_u32(top, byte == 255u ? 0u : byte);  // (a block that is not a number stays that)
        }
        top = group_max<64>(top);
        const uint32_t by = top > kFloat16Scale ? top - kFloat16Scale : 0u;
        raise = __uint_as_float((127u + by) << 23);
        if (lane == 0) shift[row] = (uint8_t)by;
    }
    const T* const from = dy + slot / top_k * H;
    float dot = 0.f;
    for (uint32_t c = 0; c < quads; ++c) {
        const uint32_t h = c * 512u + lane * 8u;
        const bool in = h < H;
        float d[8];
        uint32_t m = 0;
        if (in) {
            const Vec16<T> v = *reinterpret_cast<const Vec16<T>*>(from + h);
            Vec16<T> out;
            if (d_gates) {
                const Vec16<T> w = load_streaming16(reinterpret_cast<const Vec16<T>*>(o + row * H + h));
#pragma unroll
                for (int i = 0; i < 8; ++i) dot += Num<T>::up(v.v[i]) * Num<T>::up(w.v[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = gate * Num<T>::up(v.v[i]);
                out.v[i] = Num<T>::down(SHIFTED ? d[i] * raise : d[i]);
                m = max_u32(m, magnitude_bits(d[i]));
            }
            if (d_o) *reinterpret_cast<Vec16<T>*>(d_o + row * H + h) = out;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = 0.f;
        }
        if (values) {
            const uint32_t byte = scale_byte(group_max<16>(m));
            const float inverse = scale_inverse(byte);
            if (in) {
                uint2 q;
                q.x = pack4(d[0] * inverse, d[1] * inverse, d[2] * inverse, d[3] * inverse);
                q.y = pack4(d[4] * inverse, d[5] * inverse, d[6] * inverse, d[7] * inverse);
                *reinterpret_cast<uint2*>(values + row * H + h) = q;
            }
            uint32_t four = byte << ((lane >> 4) * 8u);
            four |= (uint32_t)__shfl_xor((int)four, 16, kWave);
            four |= (uint32_t)__shfl_xor((int)four, 32, kWave);
            if (lane == 0) scales[row * quads + c] = four;
        }
    }
    if (d_gates) {
        dot = wave_sum(dot);
        if (lane == 0) d_gates[slot] = Num<T>::down(dot);
    }
}

// ---- memory ---------------------------------------------------------------------------------------------------------

struct Buffers {
    uint8_t *x8, *x8_s, *a8, *a8_s, *h8, *h8_s;
    void* o;
    uint32_t *counts, *offsets;
    int32_t *perm, *inv;
    int64_t bytes;
};

struct Shape {
    int64_t T, k, E, H, I, R;
};

int64_t thin_output_offset(const Shape& s) { return (s.R * s.I * 4 + 255) & ~(int64_t)255; }

// The pieces of one buffer, each at a multiple of 256 bytes. keep: the pre-activation among them.
Buffers lay_out(uint8_t* base, const Shape& s, bool keep) {
    Buffers b = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) -> uint8_t* {
        uint8_t* const p = base ? base + at : nullptr;
        at += (bytes + 255) & ~(int64_t)255;
        return p;
    };
    b.x8 = take(s.T * s.H);
    b.x8_s = take(s.T * scale_pitch(s.H));
    b.a8 = take(s.R * s.I);
    b.a8_s = take(s.R * scale_pitch(s.I));
    b.o = take(s.R * s.H * 2);
    b.counts = (uint32_t*)take(s.E * 4);
    b.offsets = (uint32_t*)take(s.E * 4);
    b.perm = (int32_t*)take(s.R * 4);
    b.inv = (int32_t*)take(s.R * 4);
    if (keep) {
        b.h8 = take(s.R * 2 * s.I);
        b.h8_s = take(s.R * 2 * scale_pitch(s.I));
    }
    b.bytes = at;
    if (!keep && are_thin_experts(s.E, s.R, s.H, s.I)) {  // few rows: activation and output in fp32 take the place of all that
        const int64_t thin = thin_output_offset(s) + s.R * s.H * 4;
        if (b.bytes < thin) b.bytes = thin;
    }
    return b;
}

// the index build's scratch: the expert of every row, and its histograms
int64_t index_rows_bytes(int64_t R) { return (R * 4 + 255) & ~(int64_t)255; }

struct GradBuffers {
    uint8_t *do8, *do8_s, *dh8, *dh8_s;
    void *d_o, *dh, *dx, *a16, *x16;
    uint8_t* shift;
    int64_t bytes;
};

GradBuffers lay_out_grad(uint8_t* base, const Shape& s) {
    GradBuffers b = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) -> uint8_t* {
        uint8_t* const p = base ? base + at : nullptr;
        at += (bytes + 255) & ~(int64_t)255;
        return p;
    };
    b.do8 = take(s.R * s.H);
    b.do8_s = take(s.R * scale_pitch(s.H));
    b.d_o = take(s.R * s.H * 2);
    b.dh8 = take(s.R * 2 * s.I);
    b.dh8_s = take(s.R * 2 * scale_pitch(s.I));
    b.dh = take(s.R * 2 * s.I * 2);
    b.dx = take(s.R * s.H * 2);
    b.a16 = take(s.R * s.I * 2);
    b.x16 = take(s.T * s.H * 2);
    b.shift = take(s.R);
    b.bytes = at;
    return b;
}

int check_shape(const char* who, const Shape& s, int dtype) {
    FMA_REQUIRE(dtype == FMA_BF16 || dtype == FMA_F16, FMA_ERR_BAD_DTYPE, "%s: 16-bit tokens only, got dtype code %d", who, dtype);
    FMA_REQUIRE(s.T >= 0 && s.k >= 1 && s.E >= 1 && s.H >= 1 && s.I >= 1, FMA_ERR_BAD_SIZE, "%s: bad size T=%lld k=%lld E=%lld H=%lld I=%lld",
                who, (long long)s.T, (long long)s.k, (long long)s.E, (long long)s.H, (long long)s.I);
    FMA_REQUIRE(s.H % 16 == 0 && s.I % 16 == 0, FMA_ERR_BAD_SIZE, "%s: H=%lld and I=%lld must be multiples of 16", who, (long long)s.H, (long long)s.I);
    FMA_REQUIRE(s.k <= 65536 && s.T <= ((1ll << 31) - 1) / s.k, FMA_ERR_TOO_MANY_ELEMENTS, "%s: more than 2^31 - 1 (token, choice) slots", who);
    FMA_REQUIRE(s.I < (1 << 20) && s.H < (1 << 21) && s.T * s.H < (1ll << 30), FMA_ERR_TOO_MANY_ELEMENTS,
                "%s: I < 2^20, H < 2^21, T * H < 2^30", who);
    // (launches of one workgroup per token, of one per four slots, of a thread per 32 elements of the activation)
    FMA_REQUIRE(s.T <= kMostWorkgroups && (s.R + 3) / 4 <= kMostWorkgroups && s.R < (1ll << 37) / s.I, FMA_ERR_TOO_MANY_ELEMENTS,
                "%s: T < 2^24, T * top_k < 2^26 - 3, T * top_k * I < 2^37", who);
    if (const int rc = check_gemm(who, s.E, s.R, s.I, s.H, 2)) return rc;
    return check_gemm(who, s.E, s.R, s.H, s.I, 2);
}

}  // namespace
}  // namespace fmahip

extern "C" {

int64_t fma_swiglu_experts_fp8_buffer_bytes(int64_t T, int64_t top_k, int64_t E, int64_t H, int64_t I, int keep) {
    using namespace fmahip;
    if (T < 0 || top_k < 1 || E < 1 || H < 1 || I < 1) return 0;
    return lay_out(nullptr, Shape{T, top_k, E, H, I, T * top_k}, keep != 0).bytes;
}

int64_t fma_swiglu_experts_fp8_bwd_workspace_bytes(int64_t T, int64_t top_k, int64_t H, int64_t I) {
    using namespace fmahip;
    if (T < 0 || top_k < 1 || H < 1 || I < 1) return 0;
    return lay_out_grad(nullptr, Shape{T, top_k, 1, H, I, T * top_k}).bytes;
}

int64_t fma_swiglu_experts_fp8_workspace_bytes(int64_t T, int64_t top_k, int64_t E) {
    using namespace fmahip;
    if (T < 1 || top_k < 1 || E < 1) return 4;
    const int64_t index = fma_moe_build_index_workspace_bytes(T * top_k, E);
    return index_rows_bytes(T * top_k) + (index < 4 ? 4 : index);
}

int fma_swiglu_experts_fp8(const void* x, const void* gates, const void* ids, int id_bytes, const void* W1, const void* W1_scales,
                           const void* W2, const void* W2_scales, void* y, int64_t T, int64_t top_k, int64_t E, int64_t H, int64_t I,
                           int keep, void* buffer, int64_t buffer_bytes, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
    using namespace fmahip;
    const Shape s = {T, top_k, E, H, I, T > 0 && top_k > 0 ? T * top_k : 0};
    if (const int rc = check_shape("swiglu_experts_fp8", s, dtype)) return rc;
    if (T == 0) return FMA_OK;
    FMA_REQUIRE(x && gates && ids && W1 && W1_scales && W2 && W2_scales && y && buffer && workspace, FMA_ERR_NULL_POINTER, "swiglu_experts_fp8: a tensor is NULL");
    FMA_REQUIRE(aligned16(x) && aligned16(W1) && aligned16(W2) && aligned16(y) && aligned16(buffer) && aligned16(workspace), FMA_ERR_MISALIGNED,
                "swiglu_experts_fp8: tensors must be aligned to 16 bytes");
    FMA_REQUIRE(((reinterpret_cast<uintptr_t>(W1_scales) | reinterpret_cast<uintptr_t>(W2_scales)) & 3u) == 0, FMA_ERR_MISALIGNED,
                "swiglu_experts_fp8: scales must be aligned to 4 bytes");
    FMA_REQUIRE(id_bytes == 4 || id_bytes == 8, FMA_ERR_BAD_DTYPE, "swiglu_experts_fp8: ids must be int32 or int64");
    FMA_REQUIRE((reinterpret_cast<uintptr_t>(ids) & (uintptr_t)(id_bytes - 1)) == 0, FMA_ERR_MISALIGNED, "swiglu_experts_fp8: ids are not aligned to their size");
    const Buffers b = lay_out((uint8_t*)buffer, s, keep != 0);
    FMA_REQUIRE(buffer_bytes >= b.bytes, FMA_ERR_WORKSPACE_TOO_SMALL, "swiglu_experts_fp8: buffer of %lld bytes, %lld needed", (long long)buffer_bytes,
                (long long)b.bytes);
    const int64_t needed = fma_swiglu_experts_fp8_workspace_bytes(T, top_k, E);
    FMA_REQUIRE(workspace_bytes >= needed, FMA_ERR_WORKSPACE_TOO_SMALL, "swiglu_experts_fp8: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)needed);
    hipStream_t st = (hipStream_t)stream;
    if (!keep && are_thin_experts(E, s.R, H, I)) {
        float* const act = (float*)buffer;
        float* const o = (float*)((uint8_t*)buffer + thin_output_offset(s));
        if (const int rc = launch_thin_experts(x, ids, id_bytes, W1, W1_scales, W2, W2_scales, act, o, T, top_k, E, H, I, dtype, st)) return rc;
        return dtype == FMA_BF16 ? sum_choices<bf16_t, float>(o, ids, id_bytes, nullptr, gates, T, top_k, E, H, y, st)
                                 : sum_choices<f16_t, float>(o, ids, id_bytes, nullptr, gates, T, top_k, E, H, y, st);
    }
    if (const int rc = fma_quantize_fp8(x, b.x8, b.x8_s, nullptr, nullptr, 1, T, H, 1, dtype, stream)) return rc;
    const int64_t eid_bytes = index_rows_bytes(s.R);
    if (const int rc = fma_moe_build_index(ids, id_bytes, s.R, E, b.counts, b.offsets, b.perm, (int32_t*)workspace, b.inv,
                                           (uint8_t*)workspace + eid_bytes, workspace_bytes - eid_bytes, stream))
        return rc;
    GemmArgs a = {};
    a.A = b.x8;
    a.A_s = b.x8_s;
    a.B = (const uint8_t*)W1;
    a.B_s = (const uint8_t*)W1_scales;
    a.sizes = b.counts;
    a.row_index = b.perm;
    a.divisor = (uint32_t)top_k;
    a.a_rows = (uint32_t)T;
    a.E = (uint32_t)E;
    a.R = (uint32_t)s.R;
    a.N = (uint32_t)I;
    a.K = (uint32_t)H;
    a.segs = 1;
    a.a_pitch = (uint32_t)H;
    a.as_pitch = a.bs_pitch = (uint32_t)scale_pitch(H);
    a.b_half = (uint32_t)(I * H);
    a.bs_half = (uint32_t)((I + kBlock - 1) / kBlock * a.bs_pitch);
    a.b_group = 2 * (uint64_t)a.b_half;
    a.bs_group = 2 * (uint64_t)a.bs_half;
    a.out = b.a8;
    a.out_s = b.a8_s;
    a.h = b.h8;
    a.h_s = b.h8_s;
    a.o_pitch_s = (uint32_t)scale_pitch(I);
    if (const int rc = launch_gemm("swiglu_experts_fp8", keep ? EPI_GLU_KEEP : EPI_GLU, a, st)) return rc;
    if (const int rc = fma_grouped_gemm_fp8(b.a8, b.a8_s, W2, W2_scales, b.o, b.counts, E, s.R, H, I, dtype, stream)) return rc;
    return dtype == FMA_BF16 ? sum_choices<bf16_t>(b.o, ids, id_bytes, b.inv, gates, T, top_k, E, H, y, st)
                             : sum_choices<f16_t>(b.o, ids, id_bytes, b.inv, gates, T, top_k, E, H, y, st);
}

int fma_swiglu_experts_fp8_bwd(const void* dy, const void* gates, const void* ids, int id_bytes, const void* W1t, const void* W1t_scales, const void* W2t,
                               const void* W2t_scales, const void* buffer, int64_t buffer_bytes, void* dx, void* d_gates, void* dW1, void* dW2,
                               int64_t T, int64_t top_k, int64_t E, int64_t H, int64_t I, void* workspace, int64_t workspace_bytes, int dtype,
                               void* stream) {
    using namespace fmahip;
    const Shape s = {T, top_k, E, H, I, T > 0 && top_k > 0 ? T * top_k : 0};
    if (const int rc = check_shape("swiglu_experts_fp8_bwd", s, dtype)) return rc;
    if (T == 0) return FMA_OK;
    FMA_REQUIRE(dy && gates && ids && W1t && W1t_scales && W2t && W2t_scales && buffer && workspace, FMA_ERR_NULL_POINTER,
                "swiglu_experts_fp8_bwd: a tensor is NULL");
    FMA_REQUIRE(aligned16(dy) && aligned16(W1t) && aligned16(W2t) && aligned16(buffer) && aligned16(workspace) && aligned16(dx) && aligned16(dW1) &&
                    aligned16(dW2),
                FMA_ERR_MISALIGNED, "swiglu_experts_fp8_bwd: tensors must be aligned to 16 bytes");
    FMA_REQUIRE(((reinterpret_cast<uintptr_t>(W1t_scales) | reinterpret_cast<uintptr_t>(W2t_scales)) & 3u) == 0, FMA_ERR_MISALIGNED,
                "swiglu_experts_fp8_bwd: scales must be aligned to 4 bytes");
    FMA_REQUIRE(id_bytes == 4 || id_bytes == 8, FMA_ERR_BAD_DTYPE, "swiglu_experts_fp8_bwd: ids must be int32 or int64");
    const Buffers b = lay_out((uint8_t*)const_cast<void*>(buffer), s, true);
    FMA_REQUIRE(buffer_bytes >= b.bytes, FMA_ERR_WORKSPACE_TOO_SMALL, "swiglu_experts_fp8_bwd: buffer of %lld bytes, %lld needed", (long long)buffer_bytes,
                (long long)b.bytes);
    const GradBuffers g = lay_out_grad((uint8_t*)workspace, s);
    FMA_REQUIRE(workspace_bytes >= g.bytes, FMA_ERR_WORKSPACE_TOO_SMALL, "swiglu_experts_fp8_bwd: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)g.bytes);
    hipStream_t st = (hipStream_t)stream;
    const bool needs_h = dx || dW1;
    const dim3 grid((uint32_t)((s.R + 3) / 4)), block(kThreads);
    auto combine_bwd = [&](auto kernel, auto* dy_, auto* o_, auto* gates_, auto* d_o_, auto* d_gates_) {
        hipLaunchKernelGGL(kernel, grid, block, 0, st, dy_, o_, ids, id_bytes, b.inv, gates_, s.R, (uint32_t)top_k, (uint32_t)E, (uint32_t)H, d_o_, needs_h ? g.do8 : nullptr,
                           (uint32_t*)g.do8_s, d_gates_, b.a8_s, (uint32_t)((I + kBlock - 1) / kBlock), (uint32_t)scale_pitch(I), g.shift);
    };
    if (dtype == FMA_BF16)
        combine_bwd(combine_bwd_fp8_kernel<bf16_t, false>, (const bf16_t*)dy, (const bf16_t*)b.o, (const bf16_t*)gates, (bf16_t*)(dW2 ? g.d_o : nullptr), (bf16_t*)d_gates);
    else
        combine_bwd(dW2 ? combine_bwd_fp8_kernel<f16_t, true> : combine_bwd_fp8_kernel<f16_t, false>, (const f16_t*)dy, (const f16_t*)b.o, (const f16_t*)gates, (f16_t*)(dW2 ? g.d_o : nullptr), (f16_t*)d_gates);
    if (const int rc = launch_status("swiglu_experts_fp8_bwd")) return rc;
    if (dW2) {
        const int rc_a = dtype == FMA_BF16 ? fma_dequantize_fp8(b.a8, b.a8_s, g.a16, 1, s.R, I, 1, dtype, stream)
                                           : dequantize_shifted(b.a8, b.a8_s, g.shift, g.a16, s.R, I, st);
        if (rc_a) return rc_a;
        if (const int rc = fma_grouped_gemm_ragged(g.d_o, g.a16, dW2, b.counts, nullptr, E, /*FMA_VARY_K*/ 1, H, I, 0, 1, 0, 1.0f, dtype, stream)) return rc;
    }
    if (!needs_h) return FMA_OK;
    GemmArgs a = {};
    a.A = g.do8;
    a.A_s = g.do8_s;
    a.B = (const uint8_t*)W2t;  // [E, I, H]
    a.B_s = (const uint8_t*)W2t_scales;
    a.sizes = b.counts;
    a.E = (uint32_t)E;
    a.R = (uint32_t)s.R;
    a.N = (uint32_t)I;
    a.K = (uint32_t)H;
    a.segs = 1;
    a.a_pitch = (uint32_t)H;
    a.as_pitch = a.bs_pitch = (uint32_t)scale_pitch(H);
    a.b_group = (uint64_t)I * H;
    a.bs_group = (uint64_t)((I + kBlock - 1) / kBlock) * a.bs_pitch;
    a.D = g.dh;
    a.out = g.dh8;
    a.out_s = g.dh8_s;
    a.h = b.h8;
    a.h_s = b.h8_s;
    a.o_pitch_s = (uint32_t)scale_pitch(I);
    if (const int rc = launch_gemm("swiglu_experts_fp8_bwd", dtype == FMA_BF16 ? EPI_GLU_BWD_BF16 : EPI_GLU_BWD_F16, a, st)) return rc;
    if (dW1) {
        if (const int rc = fma_dequantize_fp8(b.x8, b.x8_s, g.x16, 1, T, H, 1, dtype, stream)) return rc;
        if (const int rc = fma_grouped_gemm_gathered_wgrad(g.dh, g.x16, T, b.perm, (int32_t)top_k, dW1, b.counts, E, 2 * I, H, 1.0f, dtype, stream)) return rc;
    }
    if (dx) {
        GemmArgs c = {};
        c.A = g.dh8;  // [R, 2, I]: the reduction in two segments
        c.A_s = g.dh8_s;
        c.B = (const uint8_t*)W1t;  // [E, 2, H, I]
        c.B_s = (const uint8_t*)W1t_scales;
        c.sizes = b.counts;
        c.E = (uint32_t)E;
        c.R = (uint32_t)s.R;
        c.N = (uint32_t)H;
        c.K = (uint32_t)I;
        c.segs = 2;
        c.a_pitch = (uint32_t)(2 * I);
        c.a_seg = (uint32_t)I;
        c.as_seg = c.bs_pitch = (uint32_t)scale_pitch(I);
        c.as_pitch = 2 * c.as_seg;
        c.b_seg = (uint32_t)(H * I);
        c.bs_seg = (uint32_t)((H + kBlock - 1) / kBlock * c.bs_pitch);
        c.b_group = 2 * (uint64_t)c.b_seg;
        c.bs_group = 2 * (uint64_t)c.bs_seg;
        c.D = g.dx;
        if (const int rc = launch_gemm("swiglu_experts_fp8_bwd", dtype == FMA_BF16 ? EPI_BF16 : EPI_F16, c, st)) return rc;
        return dtype == FMA_BF16 ? sum_choices<bf16_t>(g.dx, ids, id_bytes, b.inv, nullptr, T, top_k, E, H, dx, st)
                                 : sum_choices<f16_t>(g.dx, ids, id_bytes, b.inv, nullptr, T, top_k, E, H, dx, st);
    }
    return FMA_OK;
}

}  // extern "C"
