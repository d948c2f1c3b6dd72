// SwiGLU on a packed pre-activation [up | gate] that is kept for the backward pass in 8 bits: y = up * gate * sigmoid(gate) from the
// values as they come, and beside it the two halves in the block format (fp8_parts.h; blocks of 128 along each half); the backward pass
// reads those. HBM-bound: forward 3 16-bit values read or written and 2 bytes, backward 2 bytes and 3 values per output element, against 3
// and 5 values of the pair that keeps its input as it is; and what a training step holds in between is half.
//
// A wavefront takes 512 neighbouring output columns of a row, eight a lane: a block is 16 lanes, four scales of a half one dword.
#include "fp8_parts.h"

namespace fmahip {
namespace {
using namespace fp8;

constexpr int kThreads = 256;

// (the non-temporal hint where an access takes whole lines, in the 16-bit types: halves of lines would go one by one)
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    constexpr int V = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
        const Vec16<T>* const from = reinterpret_cast<const Vec16<T>*>(p) + i;
        const Vec16<T> v = V == 8 ? load_streaming16(from) : *from;
#pragma unroll
        for (int e = 0; e < V; ++e) f[i * V + e] = Num<T>::up(v.v[e]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    constexpr int V = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
        Vec16<T> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = Num<T>::down(f[i * V + e]);
        if constexpr (V == 8) store_streaming16(reinterpret_cast<Vec16<T>*>(p) + i, v);
        else *(reinterpret_cast<Vec16<T>*>(p) + i) = v;
    }
}
__device__ __forceinline__ uint2 pack8(const float (&f)[8], float inverse) {
    uint2 q;
    q.x = pack4(f[0] * inverse, f[1] * inverse, f[2] * inverse, f[3] * inverse);
    q.y = pack4(f[4] * inverse, f[5] * inverse, f[6] * inverse, f[7] * inverse);
    return q;
}
__device__ __forceinline__ void unpack8(uint2 q, float scale, float (&f)[8]) {
    float a[4], b[4];
    unpack4(q.x, a);
    unpack4(q.y, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = a[i] * scale;
        f[4 + i] = b[i] * scale;
    }
}
// the bytes of the four blocks of a wavefront as one dword; a block outside the row has 127
__device__ __forceinline__ uint32_t four_scales(uint32_t byte, bool in) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t four = (__shfl((int)in, (int)(lane & 48u), kWave) ? byte : 127u) << ((lane >> 4) * 8u);
    four |= (uint32_t)__shfl_xor((int)four, 16, kWave);
    return four | (uint32_t)__shfl_xor((int)four, 32, kWave);
}

// I a multiple of eight; `quads` of 512 columns per row
template <typename T, int UNROLL>
__global__ __launch_bounds__(kThreads) void swiglu_fp8_fwd_kernel(const T* __restrict__ x, T* __restrict__ y, uint8_t* __restrict__ values,
                                                                  uint32_t* __restrict__ scales, int64_t total, uint32_t quads, int64_t I) {
    const uint32_t lane = threadIdx.x & 63u;
    const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 64, step = (int64_t)gridDim.x * (kThreads / 64);
    float up[UNROLL][8], gate[UNROLL][8];
    int64_t row[UNROLL], col[UNROLL];
    bool in[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t unit = first + u * step;
        row[u] = total < (1ll << 31) ? (int64_t)((uint32_t)unit / quads) : unit / quads;
        col[u] = (unit - row[u] * quads) * 512 + lane * 8;
        in[u] = unit < total && col[u] < I;
        if (in[u]) {
            load8(x + row[u] * 2 * I + col[u], up[u]);
            load8(x + row[u] * 2 * I + I + col[u], gate[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) up[u][i] = gate[u][i] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t unit = first + u * step;
        uint32_t mu = 0, mg = 0;
        float out[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mu = max_u32(mu, magnitude_bits(up[u][i]));
            mg = max_u32(mg, magnitude_bits(gate[u][i]));
            out[i] = swiglu_f<T>(gate[u][i], up[u][i]);
        }
        const uint32_t bu = scale_byte(group_max<16>(mu)), bg = scale_byte(group_max<16>(mg));
        if (in[u]) {
            store8(y + row[u] * I + col[u], out);
            *reinterpret_cast<uint2*>(values + row[u] * 2 * I + col[u]) = pack8(up[u], scale_inverse(bu));
            *reinterpret_cast<uint2*>(values + row[u] * 2 * I + I + col[u]) = pack8(gate[u], scale_inverse(bg));
        }
        const uint32_t fu = four_scales(bu, in[u]), fg = four_scales(bg, in[u]);
        if (lane == 0 && unit < total) {
            uint32_t* const s = scales + row[u] * 2 * quads + (unit - row[u] * quads);
            s[0] = fu;
            s[quads] = fg;
        }
    }
}

template <typename T, int UNROLL>
__global__ __launch_bounds__(kThreads) void swiglu_fp8_bwd_kernel(const uint8_t* __restrict__ values, const uint8_t* __restrict__ scales,
                                                                  const T* __restrict__ dy, T* __restrict__ dx, int64_t total,
                                                                  uint32_t vectors, int64_t I, int64_t pitch) {
    // UNROLL neighbouring groups of 256 vectors of eight columns per workgroup
    const int64_t first = (int64_t)blockIdx.x * UNROLL * kThreads + threadIdx.x;
    uint2 qu[UNROLL], qg[UNROLL];
    float d[UNROLL][8], su[UNROLL], sg[UNROLL];
    int64_t row[UNROLL], col[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t v = first + u * kThreads;
        if (v < total) {
            row[u] = total < (1ll << 31) ? (int64_t)((uint32_t)v / vectors) : v / vectors;
            col[u] = (v - row[u] * vectors) * 8;
            qu[u] = *reinterpret_cast<const uint2*>(values + row[u] * 2 * I + col[u]);
            qg[u] = *reinterpret_cast<const uint2*>(values + row[u] * 2 * I + I + col[u]);
            su[u] = finite_scale_value(scales[row[u] * 2 * pitch + col[u] / kBlock]);
            sg[u] = finite_scale_value(scales[row[u] * 2 * pitch + pitch + col[u] / kBlock]);
            load8(dy + row[u] * I + col[u], d[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (first + u * kThreads < total) {
            float up[8], gate[8], du[8], dg[8];
            unpack8(qu[u], su[u], up);
            unpack8(qg[u], sg[u], gate);
#pragma unroll
            for (int i = 0; i < 8; ++i) swiglu_b<T>(gate[i], up[i], d[u][i], dg[i], du[i]);
            store8(dx + row[u] * 2 * I + col[u], du);
            store8(dx + row[u] * 2 * I + I + col[u], dg);
        }
    }
}

// any I, any alignment: eight lanes per block of 128 columns
template <typename T>
__global__ __launch_bounds__(kThreads) void swiglu_fp8_fwd_generic_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                                          uint8_t* __restrict__ values, uint8_t* __restrict__ scales,
                                                                          int64_t total, int64_t pitch, int64_t I) {
    const uint32_t lane = threadIdx.x & 7u;
    const int64_t step = (int64_t)gridDim.x * (kThreads / 8);
    for (int64_t base = (int64_t)blockIdx.x * (kThreads / 8); base < total; base += step) {
        const int64_t block = base + threadIdx.x / 8;
        const int64_t row = block / pitch, at = block - row * pitch, c0 = at * kBlock;
        const int64_t n = block < total && c0 < I ? (I - c0 < kBlock ? I - c0 : kBlock) : 0;
        const T *up = x + row * 2 * I + c0, *gate = up + I;
        uint32_t mu = 0, mg = 0;
        for (int64_t i = lane; i < n; i += 8) {
            const float u = Num<T>::up(up[i]), g = Num<T>::up(gate[i]);
            mu = max_u32(mu, magnitude_bits(u));
            mg = max_u32(mg, magnitude_bits(g));
            y[row * I + c0 + i] = Num<T>::down(swiglu_f<T>(g, u));
        }
        const uint32_t bu = scale_byte(group_max<8>(mu)), bg = scale_byte(group_max<8>(mg));
        const float iu = scale_inverse(bu), ig = scale_inverse(bg);
        for (int64_t i = lane; i < n; i += 8) {
            values[row * 2 * I + c0 + i] = (uint8_t)pack4(Num<T>::up(up[i]) * iu, 0.f, 0.f, 0.f);
            values[row * 2 * I + I + c0 + i] = (uint8_t)pack4(Num<T>::up(gate[i]) * ig, 0.f, 0.f, 0.f);
        }
        if (lane == 0 && block < total) {
            scales[row * 2 * pitch + at] = (uint8_t)(n ? bu : 127u);
            scales[row * 2 * pitch + pitch + at] = (uint8_t)(n ? bg : 127u);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void swiglu_fp8_bwd_generic_kernel(const uint8_t* __restrict__ values,
                                                                          const uint8_t* __restrict__ scales, const T* __restrict__ dy,
                                                                          T* __restrict__ dx, int64_t total, int64_t I, int64_t pitch) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
        const int64_t row = i / I, c = i - row * I;
        float u[4], g[4], dg, du;
        unpack4(values[row * 2 * I + c], u);
        unpack4(values[row * 2 * I + I + c], g);
        const float up = u[0] * finite_scale_value(scales[row * 2 * pitch + c / kBlock]);
        const float gate = g[0] * finite_scale_value(scales[row * 2 * pitch + pitch + c / kBlock]);
        swiglu_b<T>(gate, up, Num<T>::up(dy[i]), dg, du);
        dx[row * 2 * I + c] = Num<T>::down(du);
        dx[row * 2 * I + I + c] = Num<T>::down(dg);
    }
}

template <typename T>
int forward(const void* x, void* y, uint8_t* values, uint8_t* scales, int64_t R, int64_t I, hipStream_t st) {
    const int64_t pitch = scale_pitch(I);
    constexpr int kUnroll = sizeof(T) == 4 ? 1 : 2;
    const int64_t units = R * (pitch / 4), per = kUnroll * (kThreads / 64), grid = (units + per - 1) / per;
    // (2^26 and more short rows take the kernel whose workgroups make several turns)
    if (I % 8 == 0 && aligned16(x) && aligned16(y) && (reinterpret_cast<uintptr_t>(values) & 7u) == 0 && (reinterpret_cast<uintptr_t>(scales) & 3u) == 0 &&
        grid <= kMostWorkgroups) {
        hipLaunchKernelGGL((swiglu_fp8_fwd_kernel<T, kUnroll>), dim3((uint32_t)grid), dim3(kThreads), 0, st, (const T*)x, (T*)y, values,
                           (uint32_t*)scales, units, (uint32_t)(pitch / 4), I);
    } else {
        const int64_t total = R * pitch, blocks = (total + kThreads / 8 - 1) / (kThreads / 8);
        hipLaunchKernelGGL(swiglu_fp8_fwd_generic_kernel<T>, dim3((uint32_t)(blocks < (1 << 16) ? blocks : (1 << 16))), dim3(kThreads), 0, st,
                           (const T*)x, (T*)y, values, scales, total, pitch, I);
    }
    return launch_status("swiglu_fp8_forward");
}

template <typename T>
int backward(const uint8_t* values, const uint8_t* scales, const void* dy, void* dx, int64_t R, int64_t I, hipStream_t st) {
    const int64_t pitch = scale_pitch(I);
    constexpr int kUnroll = sizeof(T) == 4 ? 1 : 2;
    const int64_t vectors = R * (I / 8), per = kUnroll * kThreads, grid = (vectors + per - 1) / per;
    if (I % 8 == 0 && aligned16(dy) && aligned16(dx) && (reinterpret_cast<uintptr_t>(values) & 7u) == 0 && grid <= kMostWorkgroups) {
        hipLaunchKernelGGL((swiglu_fp8_bwd_kernel<T, kUnroll>), dim3((uint32_t)grid), dim3(kThreads), 0, st, values, scales, (const T*)dy, (T*)dx,
                           vectors, (uint32_t)(I / 8), I, pitch);
    } else {
        const int64_t total = R * I, blocks = (total + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(swiglu_fp8_bwd_generic_kernel<T>, dim3((uint32_t)(blocks < (1 << 20) ? blocks : (1 << 20))), dim3(kThreads), 0, st, values,
                           scales, (const T*)dy, (T*)dx, total, I, pitch);
    }
    return launch_status("swiglu_fp8_backward");
}

int check(const char* who, const void* a, const void* b, const void* c, const void* d, int64_t R, int64_t I, int dtype) {
    FMA_REQUIRE(dtype_bytes(dtype) != 0, FMA_ERR_BAD_DTYPE, "%s: dtype code %d", who, dtype);
    FMA_REQUIRE(R >= 0 && I >= 1, FMA_ERR_BAD_SIZE, "%s: bad size R=%lld I=%lld", who, (long long)R, (long long)I);
    FMA_REQUIRE(I <= (1ll << 31) && R <= (1ll << 40) && (R == 0 || (I + 7) / 8 <= (1ll << 38) / R), FMA_ERR_TOO_MANY_ELEMENTS, "%s: more than 2^41 elements", who);
    FMA_REQUIRE(R == 0 || (a && b && c && d), FMA_ERR_NULL_POINTER, "%s: a tensor is NULL", who);
    return FMA_OK;
}

}  // namespace
}  // namespace fmahip

extern "C" {

int fma_swiglu_fp8_forward(const void* x, void* y, void* values, void* scales, int64_t R, int64_t I, int dtype, void* stream) {
    using namespace fmahip;
    if (const int rc = check("swiglu_fp8_forward", x, y, values, scales, R, I, dtype)) return rc;
    if (R == 0) return FMA_OK;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FMA_F32) return forward<float>(x, y, (uint8_t*)values, (uint8_t*)scales, R, I, st);
    if (dtype == FMA_F16) return forward<f16_t>(x, y, (uint8_t*)values, (uint8_t*)scales, R, I, st);
    return forward<bf16_t>(x, y, (uint8_t*)values, (uint8_t*)scales, R, I, st);
}

int fma_swiglu_fp8_backward(const void* values, const void* scales, const void* dy, void* dx, int64_t R, int64_t I, int dtype, void* stream) {
    using namespace fmahip;
    if (const int rc = check("swiglu_fp8_backward", values, scales, dy, dx, R, I, dtype)) return rc;
    if (R == 0) return FMA_OK;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FMA_F32) return backward<float>((const uint8_t*)values, (const uint8_t*)scales, dy, dx, R, I, st);
    if (dtype == FMA_F16) return backward<f16_t>((const uint8_t*)values, (const uint8_t*)scales, dy, dx, R, I, st);
    return backward<bf16_t>((const uint8_t*)values, (const uint8_t*)scales, dy, dx, R, I, st);
}

}  // extern "C"
