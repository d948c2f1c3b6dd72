// Losses on the router's logits l [T, E], with the tokens that every expert is among the k choices of:
//
//   p_t = softmax(l_t),  c_e = tokens among whose k largest logits expert e is (equal logits: the lowest expert first),  N tokens counted
//   f_e = c_e / (k N),   balance = E / N sum_e f_e sum_t p_te,   z = 1 / N sum_t logsumexp(l_t)^2
//   dl_te = (g_balance E p_te (f_e - sum_i f_i p_ti) + 2 g_z logsumexp(l_t) p_te) / N
//
// A token belongs to L neighbouring lanes, each of which holds NV neighbouring logits; L * NV is the first power of two from E on, so that
// a wavefront takes 64 / L tokens at a time and a lane meets the same experts in every token: sums over tokens stay in its registers until
// the workgroup ends. Partial sums go to a workspace and are joined in a fixed order in 64 bits: the same bits on every run.
//
// The k-th largest logit is found by its bits from the top down (the largest threshold that k logits reach); the search ends where exactly
// k do. Only if logits equal to the k-th stay on both sides of the line are places among them counted.
#include "common.h"

namespace fmahip {
namespace {

constexpr int kFwdThreads = 1024, kFwdWaves = kFwdThreads / kWave;
constexpr int kBwdThreads = 256;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
struct Max {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
struct Sum {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
    static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) { return a + b; }
};
// over the L lanes of a token; every one of them gets the result
template <int L, typename OP, typename V>
__device__ __forceinline__ V over_token(V v) {
    auto as = [](V x) { return __builtin_bit_cast(uint32_t, x); };
    auto from = [](uint32_t x) { return __builtin_bit_cast(V, x); };
    if constexpr (L >= 2) v = OP::of(v, from(dpp<0xb1>(as(v))));    // the neighbour
    if constexpr (L >= 4) v = OP::of(v, from(dpp<0x4e>(as(v))));    // the other pair of the quad
    if constexpr (L >= 8) v = OP::of(v, from(dpp<0x141>(as(v))));   // the mirrored half row: the other quad
    if constexpr (L >= 16) v = OP::of(v, from(dpp<0x140>(as(v))));  // the mirrored row: its other half
    if constexpr (L >= 32) v = OP::of(v, from((uint32_t)__shfl_xor((int)as(v), 16, kWave)));
    if constexpr (L >= 64) v = OP::of(v, from((uint32_t)__shfl_xor((int)as(v), 32, kWave)));
    return v;
}

// Unsigned numbers in the order of the logits: NaN on top, -0 equal to +0; every key is above 0, which stands for "no logit here".
template <typename T>
struct Keys;
template <>
struct Keys<float> {
    static constexpr uint32_t kTop = 1u << 31;
    static __device__ __forceinline__ uint32_t of(float x) {
        uint32_t b = __float_as_uint(x);
        if (x != x) return 0xffffffffu;
        b = b == 0x80000000u ? 0u : b;
        return b & 0x80000000u ? ~b : b | 0x80000000u;
    }
};
template <typename T>
struct Keys16 {
    static constexpr uint32_t kTop = 1u << 15;
    static __device__ __forceinline__ uint32_t of(T x) {
        uint32_t b = __builtin_bit_cast(uint16_t, x);
        const float f = Num<T>::up(x);
        if (f != f) return 0xffffu;
        b = b == 0x8000u ? 0u : b;
        return b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
    }
};
template <>
struct Keys<bf16_t> : Keys16<bf16_t> {};
template <>
struct Keys<f16_t> : Keys16<f16_t> {};

template <typename T>
__device__ __forceinline__ float exp_for(float x) {
    if constexpr (sizeof(T) == 4) return expf(x);
    else return __expf(x);  // logits of 16 bits are far coarser than its error
}

// the logits of a lane: columns j * NV .. of one row; -infinity past its end
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void load_logits(const T* __restrict__ row, int first, int E, T (&x)[NV]) {
    if constexpr (VEC) {  // rows are whole 16-byte vectors
        constexpr int V = Vec16<T>::N;
#pragma unroll
        for (int i = 0; i < NV / V; ++i)
            if (first + i * V < E) {
                const Vec16<T> v = *(const Vec16<T>*)(row + first + i * V);
#pragma unroll
                for (int e = 0; e < V; ++e) x[i * V + e] = v.v[e];
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + i < E) x[i] = row[first + i];
    }
}

// softmax of a token: p (0 past its end) and, in all its lanes, the log of the sum
template <typename T, int L, int NV>
__device__ __forceinline__ float softmax_token(const T (&x)[NV], int first, int E, float (&p)[NV]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i < E) top = fmaxf(top, Num<T>::up(x[i]));
    top = over_token<L, Max>(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        p[i] = first + i < E ? exp_for<T>(Num<T>::up(x[i]) - top) : 0.f;
        sum += p[i];
    }
    sum = over_token<L, Sum>(sum);
    const float inv = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < NV; ++i) p[i] *= inv;
    return top + logf(sum);
}

// bit i of the result: whether logit i of this lane is among the token's k largest
template <typename T, int L, int NV>
__device__ __forceinline__ uint32_t choose(const T (&x)[NV], int first, int E, uint32_t k, bool counted) {
    uint32_t key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = first + i < E ? Keys<T>::of(x[i]) : 0u;
    auto reach = [&](uint32_t threshold) {
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) n += key[i] >= threshold ? 1u : 0u;
        return over_token<L, Sum>(n);
    };
    uint32_t threshold = 0;
    bool open = counted;
    for (uint32_t bit = Keys<T>::kTop; bit != 0 && __any(open); bit >>= 1) {
        const uint32_t n = reach(threshold | bit);
        if (open && n >= k) threshold |= bit;
        open = open && n != k;
    }
    uint32_t chosen = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) chosen |= (key[i] >= threshold && key[i] != 0 ? 1u : 0u) << i;
    if (__any(open)) {  // more than k reach it: those above, and of the equal ones the first
        uint32_t above = 0, equal = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            above |= (key[i] > threshold ? 1u : 0u) << i;
            equal |= (key[i] == threshold ? 1u : 0u) << i;
        }
        const uint32_t mine = __popc(equal), lane = threadIdx.x & (L - 1);
        uint32_t before = mine;  // inclusive sum over the lanes of the token
#pragma unroll
        for (int d = 1; d < L; d <<= 1) {
            const uint32_t v = (uint32_t)__shfl_up((int)before, d, L);
            before += (int)lane >= d ? v : 0u;
        }
        before -= mine;
        uint32_t left = k - over_token<L, Sum>((uint32_t)__popc(above));
        left = left > before ? left - before : 0u;  // of this lane's
        uint32_t first_ones = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t take = (equal >> i & 1u) & (left > 0 ? 1u : 0u);
            first_ones |= take << i;
            left -= take;
        }
        if (open) chosen = above | first_ones;
    }
    return counted ? chosen : 0u;
}

struct Partial {
    float* p;      // [G, E]
    uint32_t* c;   // [G, E]
    double* z;     // [G]
    uint32_t* n;   // [G]
};

template <typename T, int L, int NV, bool VEC>
__global__ __launch_bounds__(kFwdThreads) void router_loss_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask, int64_t T_,
                                                                  int E, uint32_t k, Partial part) {
    constexpr int kTokens = kFwdThreads / L;  // of a workgroup at a time
    __shared__ float s_p[kFwdWaves][L * NV];
    __shared__ uint32_t s_c[kFwdWaves][L * NV];
    __shared__ double s_z[kFwdWaves];
    __shared__ uint32_t s_n[kFwdWaves];
    const int lane = threadIdx.x & (L - 1), first = lane * NV;
    float psum[NV];
    uint32_t count[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        psum[i] = 0.f;
        count[i] = 0;
    }
    double zsum = 0.0;
    uint32_t n = 0;
    // (all lanes of a wavefront stay in the loop: they look at each other's values)
    for (int64_t base = (int64_t)blockIdx.x * kTokens; base < T_; base += (int64_t)gridDim.x * kTokens) {
        const int64_t t = base + threadIdx.x / L;
        const bool counted = t < T_ && (!mask || mask[t] != 0);
        T x[NV] = {};
        if (counted) load_logits<T, NV, VEC>(logits + t * E, first, E, x);
        float p[NV];
        const float lse = softmax_token<T, L, NV>(x, first, E, p);
        const uint32_t chosen = choose<T, L, NV>(x, first, E, k, counted);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            psum[i] += counted ? p[i] : 0.f;
            count[i] += chosen >> i & 1u;
        }
        if (counted && lane == 0) {
            zsum += (double)lse * (double)lse;
            ++n;
        }
    }
    const int wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = L; d < kWave; d <<= 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            psum[i] += __shfl_xor(psum[i], d, kWave);
            count[i] += (uint32_t)__shfl_xor((int)count[i], d, kWave);
        }
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        zsum += __shfl_xor(zsum, d, kWave);
        n += (uint32_t)__shfl_xor((int)n, d, kWave);
    }
    if ((threadIdx.x & (kWave - 1)) < L) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            s_p[wave][first + i] = psum[i];
            s_c[wave][first + i] = count[i];
        }
        if (lane == 0) {
            s_z[wave] = zsum;
            s_n[wave] = n;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kFwdThreads) {
        float p = 0.f;
        uint32_t c = 0;
#pragma unroll
        for (int w = 0; w < kFwdWaves; ++w) {
            p += s_p[w][e];
            c += s_c[w][e];
        }
        part.p[(int64_t)blockIdx.x * E + e] = p;
        part.c[(int64_t)blockIdx.x * E + e] = c;
    }
    if (threadIdx.x == 0) {
        double z = 0.0;
        uint32_t tokens = 0;
        for (int w = 0; w < kFwdWaves; ++w) {
            z += s_z[w];
            tokens += s_n[w];
        }
        part.z[blockIdx.x] = z;
        part.n[blockIdx.x] = tokens;
    }
}

// table: E f_e of every expert, then 1 / N, for the backward pass
constexpr int kJoinThreads = 1024;
__global__ __launch_bounds__(kJoinThreads) void router_loss_join_kernel(Partial part, int G, int E, uint32_t k, float* __restrict__ balance,
                                                                        float* __restrict__ z, uint32_t* __restrict__ counts,
                                                                        float* __restrict__ table) {
    __shared__ double s_sum[kJoinThreads];
    __shared__ uint64_t s_count[kJoinThreads];
    const int tid = threadIdx.x;
    auto total = [&](double v) {  // over the workgroup, in a fixed order
        s_sum[tid] = v;
        __syncthreads();
        for (int d = kJoinThreads / 2; d > 0; d >>= 1) {
            if (tid < d) s_sum[tid] += s_sum[tid + d];
            __syncthreads();
        }
        const double t = s_sum[0];
        __syncthreads();
        return t;
    };
    double zsum = 0.0, tokens = 0.0;
    for (int g = tid; g < G; g += kJoinThreads) {
        zsum += part.z[g];
        tokens += (double)part.n[g];
    }
    zsum = total(zsum);
    tokens = total(tokens);
    const double inv_n = tokens > 0.0 ? 1.0 / tokens : 0.0;
    // a power of two of columns at a time, the other threads share the rows
    int cols = 1;
    while (cols < E && cols < kJoinThreads) cols <<= 1;
    const int rows = kJoinThreads / cols, col = tid % cols, row = tid / cols;
    double p = 0.0;
    uint64_t c = 0;
    if (col < E)
        for (int g = row; g < G; g += rows) {
            p += (double)part.p[(int64_t)g * E + col];
            c += part.c[(int64_t)g * E + col];
        }
    s_sum[tid] = p;
    s_count[tid] = c;
    __syncthreads();
    for (int d = rows / 2; d > 0; d >>= 1) {
        if (row < d) {
            s_sum[tid] += s_sum[tid + d * cols];
            s_count[tid] += s_count[tid + d * cols];
        }
        __syncthreads();
    }
    p = s_sum[tid];
    c = s_count[tid];
    __syncthreads();
    double term = 0.0;
    if (row == 0 && col < E) {
        const double f = (double)c * inv_n / (double)k;
        term = f * p;
        counts[col] = (uint32_t)c;
        table[col] = (float)((double)E * f);
    }
    term = total(term);
    if (tid == 0) {
        *balance = (float)((double)E * inv_n * term);
        *z = (float)(zsum * inv_n);
        table[E] = (float)inv_n;
    }
}

template <typename T, int L, int NV, bool VEC>
__global__ __launch_bounds__(kBwdThreads) void router_loss_bwd_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask, int64_t T_,
                                                                      int E, const float* __restrict__ table,
                                                                      const float* __restrict__ balance_grad,
                                                                      const float* __restrict__ z_grad, T* __restrict__ grad) {
    constexpr int kTokens = kBwdThreads / L;
    const int first = (threadIdx.x & (L - 1)) * NV;
    const float inv_n = table[E];
    const float gb = balance_grad ? *balance_grad * inv_n : 0.f, gz = z_grad ? 2.0f * *z_grad * inv_n : 0.f;
    float f[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) f[i] = first + i < E ? table[first + i] : 0.f;
    for (int64_t base = (int64_t)blockIdx.x * kTokens; base < T_; base += (int64_t)gridDim.x * kTokens) {
        const int64_t t = base + threadIdx.x / L;
        const bool in = t < T_, counted = in && (!mask || mask[t] != 0);
        T x[NV] = {};
        if (counted) load_logits<T, NV, VEC>(logits + t * E, first, E, x);
        float p[NV];
        const float lse = softmax_token<T, L, NV>(x, first, E, p);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) dot += f[i] * p[i];
        dot = over_token<L, Sum>(dot);
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] = Num<T>::down(counted ? p[i] * (gb * (f[i] - dot) + gz * lse) : 0.f);
        if (!in) continue;
        T* const to = grad + t * E + first;
        if constexpr (VEC) {
            constexpr int V = Vec16<T>::N;
#pragma unroll
            for (int i = 0; i < NV / V; ++i)
                if (first + i * V < E) {
                    Vec16<T> v;
#pragma unroll
                    for (int e = 0; e < V; ++e) v.v[e] = x[i * V + e];
                    *(Vec16<T>*)(to + i * V) = v;
                }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (first + i < E) to[i] = x[i];
        }
    }
}

// ---- launch -----------------------------------------------------------------------------------------------------------

int64_t compute_units() { return num_compute_units() > 0 ? num_compute_units() : 256; }

int lanes_per_token(int64_t E) {
    int L = 1;
    while (L < kWave && (int64_t)L * 8 < E) L <<= 1;
    return L;
}

// workgroups of the forward pass: rows of the workspace
int64_t forward_workgroups(int64_t T, int64_t E) {
    const int64_t tokens = kFwdThreads / lanes_per_token(E), want = (T + tokens - 1) / tokens, most = compute_units();
    return want < 1 ? 1 : want < most ? want : most;
}

// calls `launch` with a token's lanes, its logits per lane, and whether rows are whole aligned vectors, as types
template <typename F>
int with_shape(int64_t E, bool vec, F launch) {
    auto as = [&](auto lanes, auto values) {
        if (vec) return launch(lanes, values, std::true_type());
        return launch(lanes, values, std::false_type());
    };
    auto eight = std::integral_constant<int, 8>();
    switch (E > 512 ? 0 : lanes_per_token(E)) {
        case 1: return as(std::integral_constant<int, 1>(), eight);
        case 2: return as(std::integral_constant<int, 2>(), eight);
        case 4: return as(std::integral_constant<int, 4>(), eight);
        case 8: return as(std::integral_constant<int, 8>(), eight);
        case 16: return as(std::integral_constant<int, 16>(), eight);
        case 32: return as(std::integral_constant<int, 32>(), eight);
        case 64: return as(std::integral_constant<int, 64>(), eight);
        default: return as(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
    }
}

template <typename T>
bool whole_vectors(const void* p, const void* q, int64_t E) {
    return aligned16(p) && aligned16(q) && E * (int64_t)sizeof(T) % 16 == 0;
}

Partial partial_of(void* workspace, int64_t G, int64_t E) {
    Partial part;
    part.z = (double*)workspace;
    part.p = (float*)(part.z + G);
    part.c = (uint32_t*)(part.p + G * E);
    part.n = part.c + G * E;
    return part;
}

template <typename T>
int launch_fwd(const void* logits, const uint8_t* mask, int64_t T_, int64_t E, int64_t k, float* balance, float* z, uint32_t* counts, float* table,
               void* workspace, hipStream_t st) {
    const int64_t G = forward_workgroups(T_, E);
    const Partial part = partial_of(workspace, G, E);
    with_shape(E, whole_vectors<T>(logits, nullptr, E), [&](auto lanes, auto values, auto vec) {
        hipLaunchKernelGGL((router_loss_kernel<T, decltype(lanes)::value, decltype(values)::value, decltype(vec)::value>), dim3((uint32_t)G),
                           dim3(kFwdThreads), 0, st, (const T*)logits, mask, T_, (int)E, (uint32_t)k, part);
        return 0;
    });
    const int rc = launch_status("router_loss");
    if (rc) return rc;
    hipLaunchKernelGGL(router_loss_join_kernel, dim3(1), dim3(kJoinThreads), 0, st, part, (int)G, (int)E, (uint32_t)k, balance, z, counts, table);
    return launch_status("router_loss (join)");
}

template <typename T>
int launch_bwd(const void* logits, const uint8_t* mask, int64_t T_, int64_t E, const float* table, const float* balance_grad, const float* z_grad,
               void* grad, hipStream_t st) {
    const int64_t tokens = kBwdThreads / lanes_per_token(E), want = (T_ + tokens - 1) / tokens, most = compute_units() * 16;
    with_shape(E, whole_vectors<T>(logits, grad, E), [&](auto lanes, auto values, auto vec) {
        hipLaunchKernelGGL((router_loss_bwd_kernel<T, decltype(lanes)::value, decltype(values)::value, decltype(vec)::value>),
                           dim3((uint32_t)(want < most ? want : most)), dim3(kBwdThreads), 0, st, (const T*)logits, mask, T_, (int)E, table,
                           balance_grad, z_grad, (T*)grad);
        return 0;
    });
    return launch_status("router_loss_bwd");
}

int check(const char* what, int64_t T, int64_t E, int dtype) {
    FMA_REQUIRE(dtype_bytes(dtype) != 0, FMA_ERR_BAD_DTYPE, "%s: unknown dtype code %d", what, dtype);
    FMA_REQUIRE(T >= 0 && T <= 0x7fffffffll, FMA_ERR_BAD_SIZE, "%s: bad number of tokens %lld", what, (long long)T);
    FMA_REQUIRE(E >= 1, FMA_ERR_BAD_SIZE, "%s: E must be at least 1 (got %lld)", what, (long long)E);
    FMA_REQUIRE(E <= FMA_MAX_GROUPS, FMA_ERR_TOO_MANY_EXPERTS, "%s: E = %lld exceeds %d", what, (long long)E, FMA_MAX_GROUPS);
    return FMA_OK;
}

}  // namespace
}  // namespace fmahip

extern "C" {

int64_t fma_router_loss_workspace_bytes(int64_t T, int64_t E) {
    if (T < 0 || E < 1 || E > FMA_MAX_GROUPS) return 0;
    return fmahip::forward_workgroups(T, E) * (8 + 4 + 8 * E);
}

int fma_router_loss(const void* logits, const uint8_t* mask, int64_t T, int64_t E, int64_t top_k, float* balance, float* z, uint32_t* counts,
                    float* table, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
    using namespace fmahip;
    const int rc = check("router_loss", T, E, dtype);
    if (rc) return rc;
    FMA_REQUIRE(top_k >= 1 && top_k <= E, FMA_ERR_BAD_SIZE, "router_loss: top_k must be in [1, %lld] (got %lld)", (long long)E, (long long)top_k);
    FMA_REQUIRE((T == 0 || logits) && balance && z && counts && table && workspace, FMA_ERR_NULL_POINTER, "router_loss: NULL pointer");
    FMA_REQUIRE(((uintptr_t)logits & (uintptr_t)(dtype_bytes(dtype) - 1)) == 0 && ((uintptr_t)workspace & 7u) == 0, FMA_ERR_MISALIGNED,
                "router_loss: logits must be aligned to their elements, the workspace to 8 bytes");
    const int64_t need = fma_router_loss_workspace_bytes(T, E);
    FMA_REQUIRE(workspace_bytes >= need, FMA_ERR_WORKSPACE_TOO_SMALL, "router_loss: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case FMA_F32: return launch_fwd<float>(logits, mask, T, E, top_k, balance, z, counts, table, workspace, st);
        case FMA_F16: return launch_fwd<f16_t>(logits, mask, T, E, top_k, balance, z, counts, table, workspace, st);
        default: return launch_fwd<bf16_t>(logits, mask, T, E, top_k, balance, z, counts, table, workspace, st);
    }
}

int fma_router_loss_bwd(const void* logits, const uint8_t* mask, int64_t T, int64_t E, const float* table, const float* balance_grad,
                        const float* z_grad, void* logits_grad, int dtype, void* stream) {
    using namespace fmahip;
    const int rc = check("router_loss_bwd", T, E, dtype);
    if (rc || T == 0) return rc;
    FMA_REQUIRE(logits && table && logits_grad, FMA_ERR_NULL_POINTER, "router_loss_bwd: NULL pointer");
    FMA_REQUIRE((((uintptr_t)logits | (uintptr_t)logits_grad) & (uintptr_t)(dtype_bytes(dtype) - 1)) == 0, FMA_ERR_MISALIGNED,
                "router_loss_bwd: tensors must be aligned to their elements");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case FMA_F32: return launch_bwd<float>(logits, mask, T, E, table, balance_grad, z_grad, logits_grad, st);
        case FMA_F16: return launch_bwd<f16_t>(logits, mask, T, E, table, balance_grad, z_grad, logits_grad, st);
        default: return launch_bwd<bf16_t>(logits, mask, T, E, table, balance_grad, z_grad, logits_grad, st);
    }
}

}  // extern "C"
