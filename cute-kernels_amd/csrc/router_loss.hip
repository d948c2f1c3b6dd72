// Losses on the router's logits l [T, E], with the tokens that every expert is among the k choices of:
//
//   p_t = softmax(l_t),  c_e = tokens among whose k largest logits expert e is (equal logits: the lowest expert first),  N tokens counted
//   f_e = c_e / (k N),   balance = E / N sum_e f_e sum_t p_te,   z = 1 / N sum_t logsumexp(l_t)^2
//   dl_te = (g_balance E p_te (f_e - sum_i f_i p_ti) + 2 g_z logsumexp(l_t) p_te) / N
//
// A token belongs to L neighbouring lanes, each of which holds NV neighbouring logits; L * NV is the first power of two from E on, so that
// a wavefront takes 64 / L tokens at a time and a lane meets the same experts in every token: sums over tokens stay in its registers until
// the workgroup ends. Partial sums go to a workspace and are joined in a fixed order in 64 bits: the same bits on every run.
#include "common.h"

#include <type_traits>

namespace fmahip {
namespace {

// threads of a workgroup of the forward pass: half of them where each holds 16 logits and would not have the registers
constexpr int fwd_threads(int values) { return values > 8 ? 512 : 1024; }
constexpr int kBwdThreads = 256;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
struct Max {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
struct Min {
    static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) { return a < b ? a : b; }
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
    if constexpr (L >= 32) {                                        // odd rows of 16 lanes and even ones
        const auto r = __builtin_amdgcn_permlane16_swap(as(v), as(v), false, false);
        v = OP::of(from((uint32_t)r[0]), from((uint32_t)r[1]));
    }
    if constexpr (L >= 64) {  // the halves of the wavefront
        const auto r = __builtin_amdgcn_permlane32_swap(as(v), as(v), false, false);
        v = OP::of(from((uint32_t)r[0]), from((uint32_t)r[1]));
    }
    return v;
}

// the sum over a wavefront's tokens: of the lanes that are the same one of their tokens
template <int L, typename V>
__device__ __forceinline__ V over_tokens(V v) {
    auto as = [](V x) { return __builtin_bit_cast(uint32_t, x); };
    auto from = [](uint32_t x) { return __builtin_bit_cast(V, x); };
    if constexpr (L <= 8) v += from(dpp<0x128>(as(v)));  // rows of 16 lanes turned by eight, four, two and one
    if constexpr (L <= 4) v += from(dpp<0x124>(as(v)));
    if constexpr (L <= 2) v += from(dpp<0x122>(as(v)));
    if constexpr (L <= 1) v += from(dpp<0x121>(as(v)));
    if constexpr (L <= 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(as(v), as(v), false, false);
        v = from((uint32_t)r[0]) + from((uint32_t)r[1]);
    }
    if constexpr (L <= 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(as(v), as(v), false, false);
        v = from((uint32_t)r[0]) + from((uint32_t)r[1]);
    }
    return v;
}

// A lane's logits as they are in memory, and widened. What is past a row's end is not fetched (a buffer's range check) and stands as -infinity:
// it adds nothing to a sum, and of equal logits the choice takes the ones further left, of which there are enough.
constexpr uint32_t kNowhere = 0x7fffffffu;
template <typename T, int NV>
struct Logits {
    static constexpr int kWords = NV * (int)sizeof(T) / 4;
    uint32_t word[kWords];
    __device__ __forceinline__ float up(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(word[i]);
        } else {
            const uint16_t bits = (uint16_t)(i & 1 ? word[i / 2] >> 16 : word[i / 2]);
            return Num<T>::up(__builtin_bit_cast(T, bits));
        }
    }
    // Zeros for a token that does not count, whatever was there; else -infinity behind the `in` logits that there are
    template <bool VEC>
    __device__ __forceinline__ void settle(bool counted, int in) {
        constexpr uint32_t kInf = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, bf16_t>::value ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
            if constexpr (sizeof(T) == 4) word[j] = j < in ? word[j] : kInf;
            else if constexpr (VEC) word[j] = 2 * j < in ? word[j] : kInf << 16 | kInf;
            else word[j] = (2 * j < in ? word[j] & 0xffffu : kInf) | (2 * j + 1 < in ? word[j] & 0xffff0000u : kInf << 16);
            word[j] = counted ? word[j] : 0u;
        }
    }
    // offset: of the lane's first logit, in bytes; `in`: how many of its logits there are
    template <bool VEC>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, uint32_t offset, int in) {
        if constexpr (VEC) {  // rows are whole 16-byte vectors
            constexpr int V = Vec16<T>::N;
#pragma unroll
            for (int v = 0; v < NV / V; ++v) {
                const auto four = __builtin_amdgcn_raw_buffer_load_b128(from, (int)(v * V < in ? offset + v * 16 : kNowhere), 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) word[v * 4 + j] = four[j];
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < NV; ++i) word[i] = __builtin_amdgcn_raw_buffer_load_b32(from, (int)(i < in ? offset + i * 4 : kNowhere), 0, 0);
        } else {
            uint32_t one[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) one[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(from, (int)(i < in ? offset + i * 2 : kNowhere), 0, 0);
#pragma unroll
            for (int i = 0; i < NV; i += 2) word[i / 2] = one[i] | one[i + 1] << 16;
        }
    }
};

// `tokens` rows of logits from p on (as many as a workgroup takes at a time, and no more than `left`) as a buffer
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const T* p, int64_t left, int tokens, int E) {
    const uint32_t rows = left > 0 ? (uint32_t)(left < tokens ? left : tokens) : 0u;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, (int)(rows * (uint32_t)E * (uint32_t)sizeof(T)), 0x00020000);
}

// the logits of a workgroup's tokens from `base` on, and whether they count (those behind the last one do not)
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void fetch_token(Logits<T, NV>& x, uint32_t& use, const T* logits, const uint8_t* mask, int64_t base, int64_t T_,
                                            int group, int E, uint32_t offset, int token, int in) {
    x.template load<VEC>(rows_at(logits + base * E, T_ - base, group, E), offset, in);
    const int64_t left = T_ - base;
    const uint32_t tokens = left > 0 ? (uint32_t)(left < group ? left : group) : 0u;
    if (mask) use = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(
                  __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(mask) + base, 0, (int)tokens, 0x00020000), token, 0, 0);
    else use = (uint32_t)token < tokens ? 1u : 0u;
}

// A token's largest logit, the exponentials of its logits against it, their sum: exp and log of the hardware, whose errors
// (two units, and that of an argument rounded in float32) are those of the subtraction in front of them.
template <typename T, int L, int NV>
__device__ __forceinline__ void softmax_token(const Logits<T, NV>& x, float (&e)[NV], float& top, float& sum) {
    top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NV; ++i) top = fmaxf(top, x.up(i));
    top = over_token<L, Max>(top);
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        e[i] = __expf(x.up(i) - top);
        sum += e[i];
    }
    sum = over_token<L, Sum>(sum);
}

// Unsigned numbers in the order of the logits: NaN on top if it is looked for, -0 equal to +0, consecutive numbers for consecutive values of the
// type; every key is above 0.
template <typename T>
struct Keys {
    static constexpr int kDrop = 0;
};
template <>
struct Keys<bf16_t> {
    static constexpr int kDrop = 16;
};
template <>
struct Keys<f16_t> {
    static constexpr int kDrop = 13;
};
template <typename T, bool NANS>
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    if constexpr (NANS) key = x != x ? 0xffffffffu : key;
    return key >> Keys<T>::kDrop;
}

// The k-th largest of a token's keys, k <= P: every lane sorts groups of P of its own downwards by comparators and keeps the P largest of two groups at
// a time, max(a_i, b_(P-1-i)), which one more pass of comparators sorts; lanes then do the same with each other's. No step depends on the values,
// and log2(L) of them go from lane to lane. For 8 of 256 that is 15 operations a logit, where a bisection takes 2 for each of its 20 to 25 steps (both
// kernels of the forward pass, us against bisection: 131072 tokens of 256 experts, 8 choices, fp32 55 / 77, bf16 57 / 77; 16384 of 1024, fp32 60 / 69;
// 65536 of 64, 6 choices, 15 / 17; 200000 of 32, 8 choices, 19 / 26). For 16 choices it was no faster (79 / 76).
__device__ __forceinline__ void order(uint32_t& larger, uint32_t& smaller) {
    const uint32_t a = larger, b = smaller;
    larger = Max::of(a, b);
    smaller = Min::of(a, b);
}
template <int P, int L, int NV>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[NV], uint32_t k) {
    uint32_t v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = key[i];
    // two sorted runs of n to one of 2 n, by Batcher's odd-even merge
#pragma unroll
    for (int n = 1; n < P; n *= 2)
#pragma unroll
        for (int run = 0; run < NV; run += 2 * n) {
#pragma unroll
            for (int i = 0; i < n; ++i) order(v[run + i], v[run + n + i]);
#pragma unroll
            for (int q = n / 2; q > 0; q /= 2)
#pragma unroll
                for (int j = q; j < 2 * n - q; j += 2 * q)
#pragma unroll
                    for (int i = 0; i < q; ++i) order(v[run + j + i], v[run + j + q + i]);
        }
    // P values that rise to their largest and fall again, or the other way round
    auto settle = [&](int at) {
#pragma unroll
        for (int d = P / 2; d > 0; d /= 2)
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (!(i & d)) order(v[at + i], v[at + i + d]);
    };
#pragma unroll
    for (int n = P; n < NV; n *= 2)
#pragma unroll
        for (int at = 0; at < NV; at += 2 * n) {
#pragma unroll
            for (int i = 0; i < P; ++i) v[at + i] = Max::of(v[at + i], v[at + n + P - 1 - i]);
            settle(at);
        }
    auto join = [&](auto other) {
        uint32_t w[P];
#pragma unroll
        for (int i = 0; i < P; ++i) w[i] = other(v[i], v[P - 1 - i]);
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = w[i];
        settle(0);
    };
    if constexpr (L >= 2) join([&](uint32_t a, uint32_t b) { return Max::of(a, dpp<0xb1>(b)); });
    if constexpr (L >= 4) join([&](uint32_t a, uint32_t b) { return Max::of(a, dpp<0x4e>(b)); });
    if constexpr (L >= 8) join([&](uint32_t a, uint32_t b) { return Max::of(a, dpp<0x141>(b)); });
    if constexpr (L >= 16) join([&](uint32_t a, uint32_t b) { return Max::of(a, dpp<0x140>(b)); });
    if constexpr (L >= 32)
        join([&](uint32_t a, uint32_t b) {
            const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false), q = __builtin_amdgcn_permlane16_swap(b, b, false, false);
            return Max::of((uint32_t)p[0], (uint32_t)q[1]);
        });
    if constexpr (L >= 64)
        join([&](uint32_t a, uint32_t b) {
            const auto p = __builtin_amdgcn_permlane32_swap(a, a, false, false), q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
            return Max::of((uint32_t)p[0], (uint32_t)q[1]);
        });
    uint32_t line = v[0];
#pragma unroll
    for (int i = 1; i < P; ++i) line = (uint32_t)i < k ? v[i] : line;
    return line;
}

// how many of a token's logits reach `line`
template <int L, int NV>
__device__ __forceinline__ uint32_t reach(const uint32_t (&key)[NV], uint32_t line) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) n += key[i] >= line ? 1u : 0u;
    return over_token<L, Sum>(n);
}

// Adds one to count[i] of the token's k largest logits, where `low` is the k-th largest, or (`exact`) exactly k reach it. Only where equal logits are
// left on both sides of the line are places among them counted.
template <int L, int NV>
__device__ __forceinline__ void count_from(const uint32_t (&key)[NV], uint32_t low, uint32_t k, bool exact, bool counted, uint32_t (&count)[NV]) {
    if (!__any(!exact)) {
        const uint32_t line = counted ? low : 0xffffffffu;
#pragma unroll
        for (int i = 0; i < NV; ++i) count[i] += key[i] >= line ? 1u : 0u;
        return;
    }
    // k or more reach it: those above, and of the equal ones the first
    uint32_t above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        above |= (key[i] > low ? 1u : 0u) << i;
        equal |= (key[i] == low ? 1u : 0u) << i;
    }
    const uint32_t mine = __popc(equal), lane = threadIdx.x & (L - 1);
    uint32_t before = mine;  // inclusive sum over the lanes of the token
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
        const uint32_t v = (uint32_t)__shfl_up((int)before, d, L);
        before += lane >= (uint32_t)d ? v : 0u;
    }
    before -= mine;
    uint32_t left = k - over_token<L, Sum>((uint32_t)__popc(above));
    left = left > before ? left - before : 0u;  // of this lane's
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t take = equal >> i & (left > 0 ? 1u : 0u);
        left -= take;
        count[i] += counted ? (above >> i & 1u) | take : 0u;
    }
}

// by the k-th largest logit itself, k <= P; no logit is a NaN
template <int P, typename T, int L, int NV>
__device__ __forceinline__ void count_sorted(const Logits<T, NV>& x, uint32_t k, bool counted, uint32_t (&count)[NV]) {
    uint32_t key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = key_of<T, false>(x.up(i));
    const uint32_t line = kth_largest<P, L, NV>(key, k);
    const bool exact = !counted || reach<L, NV>(key, line) == k;
    count_from<L, NV>(key, line, k, exact, counted, count);
}

// By bisection of the keys between the smallest of the lanes' largest (where k lanes have logits) and the largest, which ends where exactly k reach
// the middle.
template <typename T, int L, int NV, bool NANS>
__device__ __forceinline__ void count_bisected(const Logits<T, NV>& x, int in, bool enough_lanes, uint32_t k, bool counted, uint32_t (&count)[NV]) {
    uint32_t key[NV], most = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        key[i] = key_of<T, NANS>(x.up(i));
        most = Max::of(most, key[i]);
    }
    uint32_t least = most;
    if (!enough_lanes) {
#pragma unroll
        for (int i = 0; i < NV; ++i) least = Min::of(least, key[i]);
    }
    uint32_t low = over_token<L, Min>(in > 0 ? least : 0xffffffffu), high = over_token<L, Max>(most);
    bool exact = !counted;
    while (__any(!exact && low < high)) {
        const uint32_t mid = low + (high - low + 1) / 2, n = reach<L, NV>(key, mid);
        if (!exact && low < high) {
            if (n >= k) low = mid;
            else high = mid - 1;
            exact = n == k;
        }
    }
    count_from<L, NV>(key, low, k, exact, counted, count);
}

template <typename T, int L, int NV>
__device__ __forceinline__ void count_largest(const Logits<T, NV>& x, int in, bool enough_lanes, uint32_t k, bool nans, bool counted,
                                              uint32_t (&count)[NV]) {
    if (nans) count_bisected<T, L, NV, true>(x, in, enough_lanes, k, counted, count);
    else if (k <= 2) count_sorted<2, T, L, NV>(x, k, counted, count);
    else if (k <= 4) count_sorted<4, T, L, NV>(x, k, counted, count);
    else if (k <= 8) count_sorted<8, T, L, NV>(x, k, counted, count);
    else count_bisected<T, L, NV, false>(x, in, enough_lanes, k, counted, count);
}

struct Partial {
    float* p;      // [G, E]
    uint32_t* c;   // [G, E]
    double* z;     // [G]
    uint32_t* n;   // [G]
    double* term;  // what each workgroup of the join contributes to the balance
};

// Bound by vector instructions where there are many choices and logits: 131072 tokens of 256 experts, 8 choices, take 46 to 49 us (fp32, 2.8 TB/s;
// bf16 47 to 51), 35 instructions a logit (bf16 38) that issue in 70 % of the cycles of two wavefronts per SIMD. Three of them (768 threads) gain 5 %
// there, 10 % with 16 choices, and lose 3 % with 160 or 161 experts, whose registers no longer suffice. With two choices this kernel and the join
// take 46 us, with eight 59, with sixteen 79.
template <typename T, int L, int NV, bool VEC>
__global__ __launch_bounds__(fwd_threads(NV)) void router_loss_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask, int64_t T_,
                                                                  int E, uint32_t k, Partial part) {
    constexpr int kFwdThreads = fwd_threads(NV), kFwdWaves = kFwdThreads / kWave, kTokens = kFwdThreads / L;  // tokens of a workgroup at a time
    __shared__ float s_p[kFwdWaves][L * NV];
    __shared__ uint32_t s_c[kFwdWaves][L * NV];
    __shared__ double s_z[kFwdWaves];
    __shared__ uint32_t s_n[kFwdWaves];
    const int lane = threadIdx.x & (L - 1), first = lane * NV, token = threadIdx.x / L;
    const int in = E - first < 0 ? 0 : E - first < NV ? E - first : NV;
    const bool enough_lanes = (uint32_t)((E + NV - 1) / NV) >= k;
    const uint32_t offset = (uint32_t)(token * E + first) * (uint32_t)sizeof(T);
    float psum[NV];
    uint32_t count[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        psum[i] = 0.f;
        count[i] = 0;
    }
    double zsum = 0.0;
    uint32_t n = 0;
    auto fetch = [&](Logits<T, NV>& x, uint32_t& use, int64_t base) {
        fetch_token<T, NV, VEC>(x, use, logits, mask, base, T_, kTokens, E, offset, token, in);
    };
    Logits<T, NV> x, next;
    uint32_t use, next_use;
    int64_t base = (int64_t)blockIdx.x * kTokens;
    const int64_t step = (int64_t)gridDim.x * kTokens;
    fetch(x, use, base);
    // (all lanes of a wavefront stay in the loop: they look at each other's values)
    for (; base < T_; base += step) {
        fetch(next, next_use, base + step);  // the next tokens, before these are worked on
        const bool counted = use != 0;
        x.template settle<VEC>(counted, in);
        float e[NV], top, sum;
        softmax_token<T, L, NV>(x, e, top, sum);
        const float inv = counted ? __builtin_amdgcn_rcpf(sum) : 0.f, lse = counted ? top + __logf(sum) : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) psum[i] += e[i] * inv;
        zsum = __builtin_fma((double)lse, (double)lse, zsum);
        n += counted ? 1u : 0u;
        count_largest<T, L, NV>(x, in, enough_lanes, k, __any(lse != lse), counted, count);
        x = next;
        use = next_use;
    }
    if (lane != 0) {  // (the lanes of a token have the same)
        zsum = 0.0;
        n = 0;
    }
    const int wave = threadIdx.x / kWave;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        psum[i] = over_tokens<L>(psum[i]);
        count[i] = over_tokens<L>(count[i]);
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

// A workgroup joins the columns of `cols` experts (a power of two). One that has them all also forms the losses; of several each leaves its part of
// the balance to router_loss_finish_kernel. table: E f_e of every expert, then 1 / N, for the backward pass.
constexpr int kJoinThreads = 1024, kJoinWaves = kJoinThreads / kWave;
struct Total {
    double a, b;
};
// over the workgroup, in a fixed order; every thread gets both
__device__ __forceinline__ Total join_total(double a, double b, double (*slots)[2]) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        a += __shfl_xor(a, d, kWave);
        b += __shfl_xor(b, d, kWave);
    }
    if ((threadIdx.x & (kWave - 1)) == 0) {
        slots[threadIdx.x / kWave][0] = a;
        slots[threadIdx.x / kWave][1] = b;
    }
    __syncthreads();
    Total t{0.0, 0.0};
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
        t.a += slots[w][0];
        t.b += slots[w][1];
    }
    return t;
}

__global__ __launch_bounds__(kJoinThreads) void router_loss_join_kernel(Partial part, int G, int E, int cols, uint32_t k, float* __restrict__ balance,
                                                                        float* __restrict__ z, uint32_t* __restrict__ counts,
                                                                        float* __restrict__ table) {
    __shared__ double s_sum[kJoinThreads];
    __shared__ uint32_t s_count[kJoinThreads];
    __shared__ double s_total[2][kJoinWaves][2];
    // the threads of a column share its rows; eight rows of a thread on the way at a time
    const int tid = threadIdx.x, rows = kJoinThreads / cols, col = blockIdx.x * cols + (tid & (cols - 1)), row = tid / cols;
    double p = 0.0;
    uint32_t c = 0;
    if (col < E)
        for (int g = row; g < G; g += 8 * rows) {
            float pv[8];
            uint32_t cv[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int at = g + u * rows < G ? g + u * rows : g;
                pv[u] = part.p[(int64_t)at * E + col];
                cv[u] = part.c[(int64_t)at * E + col];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (g + u * rows < G) {
                    p += (double)pv[u];
                    c += cv[u];
                }
        }
    double zsum = 0.0, tokens = 0.0;
    if (tid < G) {  // (G is at most the number of compute units)
        zsum = part.z[tid];
        tokens = (double)part.n[tid];
    }
    const Total all = join_total(zsum, tokens, s_total[0]);
    const double inv_n = all.b > 0.0 ? 1.0 / all.b : 0.0;
    s_sum[tid] = p;
    s_count[tid] = c;
    __syncthreads();
    double term = 0.0;
    if (tid < cols && col < E) {
        for (int r = 1; r < rows; ++r) {
            p += s_sum[tid + r * cols];
            c += s_count[tid + r * cols];
        }
        const double f = (double)c * inv_n / (double)k;
        term = f * p;
        counts[col] = c;
        table[col] = (float)((double)E * f);
    }
    const Total loss = join_total(term, 0.0, s_total[1]);
    if (tid != 0) return;
    part.term[blockIdx.x] = (double)E * inv_n * loss.a;
    if (gridDim.x > 1) return;
    *balance = (float)part.term[0];
    *z = (float)(all.a * inv_n);
    table[E] = (float)inv_n;
}

__global__ __launch_bounds__(kWave) void router_loss_finish_kernel(Partial part, int G, int E, int joins, float* __restrict__ balance,
                                                                   float* __restrict__ z, float* __restrict__ table) {
    double loss = (int)threadIdx.x < joins ? part.term[threadIdx.x] : 0.0, zsum = 0.0, tokens = 0.0;
    for (int g = threadIdx.x; g < G; g += kWave) {
        zsum += part.z[g];
        tokens += (double)part.n[g];
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        loss += __shfl_xor(loss, d, kWave);
        zsum += __shfl_xor(zsum, d, kWave);
        tokens += __shfl_xor(tokens, d, kWave);
    }
    if (threadIdx.x != 0) return;
    const double inv_n = tokens > 0.0 ? 1.0 / tokens : 0.0;
    *balance = (float)loss;
    *z = (float)(zsum * inv_n);
    table[E] = (float)inv_n;
}

// One pass over logits and gradient, the softmax formed again. HBM-bound from some megabytes on: 131072 tokens of 256 experts in fp32 take 53 us, 5.0
// TB/s, with logits from memory, and 43 behind a forward pass that left part of them in the last-level cache; in bf16 29 us, 4.6 TB/s, where vector
// instructions come near the bound as well (26 a logit); 32768 of 128 in bf16 take 7 us, of which a launch is 5.
template <typename T, int L, int NV, bool VEC>
__global__ __launch_bounds__(kBwdThreads) void router_loss_bwd_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask, int64_t T_,
                                                                      int E, const float* __restrict__ table,
                                                                      const float* __restrict__ balance_grad,
                                                                      const float* __restrict__ z_grad, T* __restrict__ grad) {
    constexpr int kTokens = kBwdThreads / L;
    const int first = (threadIdx.x & (L - 1)) * NV, token = threadIdx.x / L;
    const int in = E - first < 0 ? 0 : E - first < NV ? E - first : NV;
    const uint32_t offset = (uint32_t)(token * E + first) * (uint32_t)sizeof(T);
    Logits<T, NV> x;
    uint32_t use;
    int64_t base = (int64_t)blockIdx.x * kTokens;
    // the first token's logits and the table's entries under way together (no branch between them); zeros behind the table's end
    fetch_token<T, NV, VEC>(x, use, logits, mask, base, T_, kTokens, E, offset, token, in);
    float f[NV];
    const __amdgpu_buffer_rsrc_t entries = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(table), 0, E * 4, 0x00020000);
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
        const auto four = __builtin_amdgcn_raw_buffer_load_b128(entries, (first + i) * 4, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t one = four[j];
            f[i + j] = __uint_as_float(one);
        }
    }
    const float inv_n = table[E];
    const float gb = balance_grad ? *balance_grad * inv_n : 0.f, gz = z_grad ? 2.0f * *z_grad * inv_n : 0.f;
    for (; base < T_; base += (int64_t)gridDim.x * kTokens) {
        const bool counted = use != 0;
        x.template settle<VEC>(counted, in);
        float e[NV], top, sum;
        softmax_token<T, L, NV>(x, e, top, sum);
        const float inv = counted ? __builtin_amdgcn_rcpf(sum) : 0.f, lse = top + __logf(sum);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            e[i] *= inv;
            dot += f[i] * e[i];
        }
        const float shift = gz * lse - gb * over_token<L, Sum>(dot);
#pragma unroll
        for (int i = 0; i < NV; ++i) e[i] = counted ? e[i] * (gb * f[i] + shift) : 0.f;
        const __amdgpu_buffer_rsrc_t to = rows_at(grad + base * E, T_ - base, kTokens, E);
        if constexpr (VEC) {
            constexpr int V = Vec16<T>::N;
#pragma unroll
            for (int v = 0; v < NV / V; ++v) {
                Vec16<T> o;
#pragma unroll
                for (int i = 0; i < V; ++i) o.v[i] = Num<T>::down(e[v * V + i]);
                typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), to, (int)(v * V < in ? offset + v * 16 : kNowhere), 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t at = i < in ? offset + (uint32_t)(i * sizeof(T)) : kNowhere;
                if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(e[i]), to, (int)at, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, Num<T>::down(e[i])), to, (int)at, 0, 0);
            }
        }
        fetch_token<T, NV, VEC>(x, use, logits, mask, base + (int64_t)gridDim.x * kTokens, T_, kTokens, E, offset, token, in);
    }
}

// ---- launch -----------------------------------------------------------------------------------------------------------

int64_t compute_units() { return num_compute_units() > 0 ? num_compute_units() : 256; }

// Logits per lane: 16 where eight would take more than a wavefront, and in the forward pass from 33 on, whose sorting and sums then need one step
// less between lanes (8 choices, both kernels of the forward pass, us against eight a lane: 131072 tokens of 256 experts, fp32 57 / 69; of 128, bf16
// 33 / 35; of 64, fp32 20 / 21. The backward pass of the first, its logits from memory: 64 / 53, of 65536 of 160, fp16, 13 / 15).
int values_per_lane(int64_t E, bool forward) { return E > (forward ? 32 : 512) ? 16 : 8; }
int lanes_per_token(int64_t E, bool forward) {
    int L = 1;
    while ((int64_t)L * values_per_lane(E, forward) < E) L <<= 1;
    return L;
}

// workgroups of the forward pass: rows of the workspace
int64_t forward_workgroups(int64_t T, int64_t E) {
    const int64_t tokens = fwd_threads(values_per_lane(E, true)) / lanes_per_token(E, true), want = (T + tokens - 1) / tokens, most = compute_units();
    return want < 1 ? 1 : want < most ? want : most;
}

template <int N>
using Int = std::integral_constant<int, N>;
// calls `launch` with a token's lanes, its logits per lane, and whether rows are whole aligned vectors, as types
template <bool FORWARD, typename F>
void with_shape(int64_t E, bool vec, F launch) {
    auto as = [&](auto lanes, auto values) {
        if (vec) launch(lanes, values, std::true_type());
        else launch(lanes, values, std::false_type());
    };
    const int L = lanes_per_token(E, FORWARD);
    if (values_per_lane(E, FORWARD) == 16) {
        if constexpr (FORWARD) {
            if (L == 4) return as(Int<4>(), Int<16>());
            if (L == 8) return as(Int<8>(), Int<16>());
            if (L == 16) return as(Int<16>(), Int<16>());
            if (L == 32) return as(Int<32>(), Int<16>());
        }
        return as(Int<64>(), Int<16>());
    }
    if (L == 1) return as(Int<1>(), Int<8>());
    if (L == 2) return as(Int<2>(), Int<8>());
    if constexpr (!FORWARD) {
        if (L == 8) return as(Int<8>(), Int<8>());
        if (L == 16) return as(Int<16>(), Int<8>());
        if (L == 32) return as(Int<32>(), Int<8>());
        if (L == 64) return as(Int<64>(), Int<8>());
    }
    return as(Int<4>(), Int<8>());
}

template <typename T>
bool whole_vectors(const void* p, const void* q, int64_t E) {
    return aligned16(p) && aligned16(q) && E * (int64_t)sizeof(T) % 16 == 0;
}

// Columns that a workgroup joins: all, or 16 (64 bytes of each row) where a single one would have more than a compute unit's loads bring in some
// microseconds, against one launch more (all of the forward pass, us one / several: 1024 experts, 256 rows 60 / 39.5, 128 rows 24.9 / 15.8; 512, 256 rows
// 34 / 26; 256, 256 rows 55.2 / 54.5; 128, 256 rows 16.9 / 19.1; 256, 64 rows 11.9 / 15.6).
constexpr int kJoinColumns = 16, kMostJoins = FMA_MAX_GROUPS / kJoinColumns;
static_assert(kMostJoins <= kWave, "router_loss_finish_kernel has a lane for each");
int join_columns(int64_t G, int64_t E) {
    int cols = 1;
    while (cols < E) cols <<= 1;
    return cols > kJoinColumns && G * cols > 64 * kJoinThreads ? kJoinColumns : cols;
}

Partial partial_of(void* workspace, int64_t G, int64_t E) {
    Partial part;
    part.z = (double*)workspace;
    part.term = part.z + G;
    part.p = (float*)(part.term + kMostJoins);
    part.c = (uint32_t*)(part.p + G * E);
    part.n = part.c + G * E;
    return part;
}

template <typename T>
int launch_fwd(const void* logits, const uint8_t* mask, int64_t T_, int64_t E, int64_t k, float* balance, float* z, uint32_t* counts, float* table,
               void* workspace, hipStream_t st) {
    const int64_t G = forward_workgroups(T_, E);
    const Partial part = partial_of(workspace, G, E);
    with_shape<true>(E, whole_vectors<T>(logits, nullptr, E), [&](auto lanes, auto values, auto vec) {
        hipLaunchKernelGGL((router_loss_kernel<T, decltype(lanes)::value, decltype(values)::value, decltype(vec)::value>), dim3((uint32_t)G),
                           dim3(fwd_threads(decltype(values)::value)), 0, st, (const T*)logits, mask, T_, (int)E, (uint32_t)k, part);
    });
    const int rc = launch_status("router_loss");
    if (rc) return rc;
    const int cols = join_columns(G, E), joins = ((int)E + cols - 1) / cols;
    hipLaunchKernelGGL(router_loss_join_kernel, dim3((uint32_t)joins), dim3(kJoinThreads), 0, st, part, (int)G, (int)E, cols, (uint32_t)k, balance, z,
                       counts, table);
    if (joins > 1) hipLaunchKernelGGL(router_loss_finish_kernel, dim3(1), dim3(kWave), 0, st, part, (int)G, (int)E, joins, balance, z, table);
    return launch_status("router_loss (join)");
}

template <typename T>
int launch_bwd(const void* logits, const uint8_t* mask, int64_t T_, int64_t E, const float* table, const float* balance_grad, const float* z_grad,
               void* grad, hipStream_t st) {
    const int64_t tokens = kBwdThreads / lanes_per_token(E, false), want = (T_ + tokens - 1) / tokens, most = compute_units() * 16;
    with_shape<false>(E, whole_vectors<T>(logits, grad, E), [&](auto lanes, auto values, auto vec) {
        hipLaunchKernelGGL((router_loss_bwd_kernel<T, decltype(lanes)::value, decltype(values)::value, decltype(vec)::value>),
                           dim3((uint32_t)(want < most ? want : most)), dim3(kBwdThreads), 0, st, (const T*)logits, mask, T_, (int)E, table,
                           balance_grad, z_grad, (T*)grad);
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
    return fmahip::forward_workgroups(T, E) * (8 + 4 + 8 * E) + 8 * fmahip::kMostJoins;
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
