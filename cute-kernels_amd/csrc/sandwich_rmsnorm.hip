// The norm behind a block, its gate and residual scale, the residual stream and the norm before the next block, forward and backward:
//
//   n   = x inv_x w_post            inv_x = 1 / sqrt(mean(x^2) + eps)
//   r   = residual + a gate n       (stored rounded; a: the residual scale)
//   out = r inv_r w                 inv_r = 1 / sqrt(mean(r^2) + eps), from the unrounded r
//
// with x^ = x inv_x, r^ = r inv_r, g = dout w:
//
//   dr = dr_in + inv_r (g - r^ mean(g r^))                      dresidual = dr
//   dgate = a dr w_post x^, summed over the rows that share it  u = a dr gate w_post
//   dx = inv_x (u - x^ mean(u x^))
//   dw = sum over rows of dout r^                               dw_post = sum over rows of a dr gate x^
//
// A gate is [G, H] or [G, 1]: every row of it serves B / G neighbouring rows of x. Sums over rows are kept by a workgroup over all of its
// rows in 32 bits; the partial sums go to a workspace and are added in a fixed order in 64 bits: the same bits on every run.
#include "common.h"

#include <initializer_list>

namespace fmahip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// Threads of the forward pass per compute unit, each with its share of a row and of the next one. us with 512 / 1024 / 2048, inputs from memory, bf16:
// [16384, 4096] 116 / 89 / 99, [16384, 2048] 51 / 51 / 51, [8188, 2880] with a full gate 57 / 41 / 45; fp32 [16384, 4096] - / 195 / 186, the least of 27
// launches 181 / 182. Within a training step, which leaves part of a row's tensors in the last-level cache, the first is 96 / 98 (the least 86 / 96) with
// 1024 / 2048, the third 41 / 45. A workgroup per row, which ends with it, took 110, 60 and 63.
constexpr int kFwdThreadsPerCU = 1024;
// teams of a workgroup: those of one wavefront meet at no barrier, four of them make a workgroup
constexpr int teams_of(int team) { return team == kWave ? 4 : 1; }
// Teams of the backward pass per compute unit, each with a row in its registers and one on the way: 512 threads. More of them add partial sums
// and gain no rate (us with a third / half / all of 1536 threads, bf16: [16384, 4096] 133 / 145 / 145, [16384, 2048] 78 / 73 / 81,
// [8188, 2880] 53 / 58 / 66, [32768, 512] 40 / 45 / -), and at least two rows for each ([300, 4096] 13.5 / 11.9 / 12.9 us with one / two / four,
// [1021, 2048] 14.6 / 15.1 / 13.6).
constexpr int workers_per_cu(int team) { return team < 512 ? 512 / team : 1; }
constexpr int kBwdMinRows = 2;

// how rows of x share a row of the gate; decides what is summed for its gradient
enum Mode {
    kNoGate,
    kFull,     // a gate row per row: its gradient is written with the row
    kChannel,  // one gate row: dgate = w_post s, dw_post = gate s with s = sum of a dr x^
    kGroup,    // some gate rows: s for each of them
    kScalar,   // one number per gate row
};

struct Shape {
    int64_t B, H;
    int64_t R;  // rows of x per gate row
    Mode mode;
};

Shape shape_of(int64_t B, int64_t H, int64_t gate_rows, int64_t gate_width) {
    Shape s{B, H, B, kNoGate};
    if (gate_rows > 0) {
        s.R = gate_rows < B ? B / gate_rows : 1;
        s.mode = gate_width < H ? kScalar : gate_rows == B ? kFull : gate_rows == 1 ? kChannel : kGroup;
    }
    return s;
}

// The workers of the backward pass: `parts` for each of `groups` of neighbouring rows (one group unless the gate has several rows that
// serve several rows each), or, with more groups than workers are wanted, whole groups for each.
struct Split {
    int64_t groups, rows, parts, workers;
    int64_t sums;  // rows of partial sums: workgroups
};
Split split_of(const Shape& s, int team, int teams) {
    const int64_t cus = num_compute_units() > 0 ? num_compute_units() : 256;
    int64_t want = cus * workers_per_cu(team);
    if (want > s.B / kBwdMinRows) want = s.B / kBwdMinRows > 0 ? s.B / kBwdMinRows : 1;
    Split p{1, s.B, 1, 1, 1};
    if (s.mode == kGroup) {
        p.groups = s.B / s.R;
        p.rows = s.R;
    }
    p.parts = want / p.groups;
    if (p.parts > p.rows) p.parts = p.rows;
    if (p.parts < 1) p.parts = 1;
    p.workers = p.parts > 1 || p.groups <= want ? p.groups * p.parts : want;
    p.sums = (p.workers + teams - 1) / teams;
    return p;
}

// the workspace: partial sums [sums, H] for dw and dw_post, [workers, H] for dgate (kGroup), one number per row (kScalar)
struct Partial {
    float *w, *wp, *gate, *rows;
};
Partial partial_of(void* workspace, const Shape& s, const Split& p) {
    Partial part;
    part.w = (float*)workspace;
    part.wp = part.w + p.sums * s.H;
    part.gate = part.rows = part.wp + p.sums * s.H;  // (never both)
    return part;
}
// enough for every type and alignment (teams of a wavefront hold rows of up to 1024 elements)
int64_t workspace_bytes_of(const Shape& s) {
    int64_t most = 0;
    for (int team : {64, 256, 1024}) {
        if (team == 64 && s.H > 1024) continue;
        const Split p = split_of(s, team, teams_of(team));
        const int64_t n = p.sums * s.H * 2 + (s.mode == kGroup ? p.workers * s.H : 0) + (s.mode == kScalar ? s.B : 0);
        most = n > most ? n : most;
    }
    return 4 * most;
}

__device__ __forceinline__ float inverse_rms(float sum_of_squares, float inv_H, float eps) {
    return 1.0f / sqrtf(sum_of_squares * inv_H + eps);
}

// Sum over the workgroup; two alternating LDS areas, so that one barrier per use is enough
__device__ __forceinline__ float workgroup_sum(float v, float (*slots)[kWaves], int& parity) {
    float* const slot = slots[parity];
    parity ^= 1;
    v = wave_sum(v);
    if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += slot[w];
    return t;
}

template <typename T>
struct FwdArgs {
    const T *x, *residual, *post_weight, *weight, *gate;
    T *out, *stream;
    float* stats;  // inv_x of every row, then inv_r; or NULL
    Shape s;
    float inv_H, eps, a;
};

template <typename T>
struct BwdArgs {
    const T *x, *residual, *post_weight, *weight, *gate, *d_out, *d_stream;
    const float* stats;
    T *dx, *d_residual, *d_gate;
    Partial part;
    Shape s;
    Split p;
    float inv_H, a;
    bool sums_w, sums_wp;  // whether the weights' gradients are wanted
};

template <typename T>
__device__ __forceinline__ float at(const T* p, int64_t i) {
    return p ? Num<T>::up(p[i]) : 1.0f;
}

__device__ __forceinline__ int64_t gate_row(const Shape& s, int64_t row) { return (uint32_t)row / (uint32_t)s.R; }  // (both below 2^31)

// ---- rows that no team holds: element by element, inputs read again from the caches ---------------------------------------------
// bf16 [2000, 20000]: forward 351 us, backward 1.8 ms (0.9 and 0.3 TB/s).

template <typename T>
__global__ __launch_bounds__(kThreads) void sandwich_fwd_generic_kernel(const FwdArgs<T> k) {
    __shared__ float s_red[2][kWaves];
    int parity = 0;
    const int64_t H = k.s.H;
    for (int64_t row = blockIdx.x; row < k.s.B; row += gridDim.x) {
        const int64_t base = row * H;
        const T* const gate = k.gate ? k.gate + gate_row(k.s, row) * (k.s.mode == kScalar ? 1 : H) : nullptr;
        const bool scalar = k.s.mode == kScalar;
        auto stream = [&](int64_t h, float inv_x) {
            const float n = Num<T>::up(k.x[base + h]) * inv_x * at(k.post_weight, h);
            return Num<T>::up(k.residual[base + h]) + k.a * (n * at(gate, scalar ? 0 : h));
        };
        float ss = 0.f;
        for (int64_t h = threadIdx.x; h < H; h += kThreads) {
            const float x = Num<T>::up(k.x[base + h]);
            ss += x * x;
        }
        const float inv_x = inverse_rms(workgroup_sum(ss, s_red, parity), k.inv_H, k.eps);
        ss = 0.f;
        for (int64_t h = threadIdx.x; h < H; h += kThreads) {
            const float r = stream(h, inv_x);
            ss += r * r;
        }
        const float inv_r = inverse_rms(workgroup_sum(ss, s_red, parity), k.inv_H, k.eps);
        for (int64_t h = threadIdx.x; h < H; h += kThreads) {
            const float r = stream(h, inv_x);
            k.stream[base + h] = Num<T>::down(r);
            k.out[base + h] = Num<T>::down(r * inv_r * at(k.weight, h));
        }
        if (k.stats && threadIdx.x == 0) {
            k.stats[row] = inv_x;
            k.stats[k.s.B + row] = inv_r;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sandwich_bwd_generic_kernel(const BwdArgs<T> k) {
    __shared__ float s_red[2][kWaves];
    int parity = 0;
    const int64_t H = k.s.H, slot = (int64_t)blockIdx.x * H;
    // column h of this workgroup's partial sums belongs to thread h % 256
    float* const w = k.sums_w ? k.part.w + slot : nullptr;
    float* const wp = k.sums_wp ? k.part.wp + slot : nullptr;
    float* const sg = k.s.mode == kGroup && k.d_gate ? k.part.gate + slot : nullptr;
    for (int64_t h = threadIdx.x; h < H; h += kThreads) {
        if (w) w[h] = 0.f;
        if (wp) wp[h] = 0.f;
    }
    const int64_t first = blockIdx.x / k.p.parts, part = blockIdx.x % k.p.parts, step = gridDim.x / k.p.parts;
    for (int64_t group = first; group < k.p.groups; group += step) {
        if (sg)
            for (int64_t h = threadIdx.x; h < H; h += kThreads) sg[h] = 0.f;
        for (int64_t i = part; i < k.p.rows; i += k.p.parts) {
            const int64_t row = group * k.p.rows + i, base = row * H;
            const bool scalar = k.s.mode == kScalar;
            const T* const gate = k.gate ? k.gate + gate_row(k.s, row) * (scalar ? 1 : H) : nullptr;
            const float inv_x = k.stats[row], inv_r = k.stats[k.s.B + row];
            auto normed = [&](int64_t h) {  // r^
                const float n = Num<T>::up(k.x[base + h]) * inv_x * at(k.post_weight, h);
                return (Num<T>::up(k.residual[base + h]) + k.a * (n * at(gate, scalar ? 0 : h))) * inv_r;
            };
            float dot = 0.f;
            if (k.d_out)
                for (int64_t h = threadIdx.x; h < H; h += kThreads)
                    dot += Num<T>::up(k.d_out[base + h]) * at(k.weight, h) * normed(h);
            const float c_r = workgroup_sum(dot, s_red, parity) * k.inv_H;
            auto d_stream = [&](int64_t h) {
                float d = k.d_stream ? Num<T>::up(k.d_stream[base + h]) : 0.f;
                if (k.d_out) d += inv_r * (Num<T>::up(k.d_out[base + h]) * at(k.weight, h) - normed(h) * c_r);
                return d;
            };
            dot = 0.f;
            float gate_dot = 0.f;
            for (int64_t h = threadIdx.x; h < H; h += kThreads) {
                const float v = k.a * d_stream(h) * at(k.post_weight, h) * Num<T>::up(k.x[base + h]);
                dot += v * at(gate, scalar ? 0 : h);
                gate_dot += v;
            }
            const float c_x = workgroup_sum(dot, s_red, parity) * inv_x * k.inv_H;
            if (scalar && k.d_gate) {
                gate_dot = workgroup_sum(gate_dot, s_red, parity) * inv_x;
                if (threadIdx.x == 0) {
                    if (k.s.R == 1) k.d_gate[row] = Num<T>::down(gate_dot);
                    else k.part.rows[row] = gate_dot;
                }
            }
            for (int64_t h = threadIdx.x; h < H; h += kThreads) {
                const float dr = d_stream(h), dz = k.a * dr, x = Num<T>::up(k.x[base + h]) * inv_x;
                const float g = at(gate, scalar ? 0 : h), p = at(k.post_weight, h);
                k.d_residual[base + h] = Num<T>::down(dr);
                k.dx[base + h] = Num<T>::down(inv_x * (dz * g * p - x * c_x));
                if (k.s.mode == kFull && k.d_gate) k.d_gate[base + h] = Num<T>::down(dz * p * x);
                if (w) w[h] += k.d_out ? Num<T>::up(k.d_out[base + h]) * normed(h) : 0.f;
                if (wp) wp[h] += k.s.mode == kChannel ? dz * x : dz * g * x;
                if (sg) sg[h] += dz * x;
            }
        }
        if (sg && k.p.parts == 1)
            for (int64_t h = threadIdx.x; h < H; h += kThreads) k.d_gate[group * H + h] = Num<T>::down(at(k.post_weight, h) * sg[h]);
    }
}

// ---- a row in the registers of its team of threads ------------------------------------------------------------------------------
//
// A team of TEAM threads per row, VPT vectors of 16 bytes per thread, the next row requested before this one is worked on. All accesses of
// the loops are buffer instructions, whose range check stands for every condition: past the row's end (each dword of an access by itself),
// behind the last row, where a tensor is absent (num_records 0), loads give zeros and stores go nowhere. A branch around a load or a store
// would make the compiler wait for everything that is outstanding, the next row included, since it cannot count what lies behind.
// Rows that start on a dword boundary are accessed 16 bytes at a time; those of an odd number of 16-bit elements, or off such a boundary,
// element by element (ELEM), in the same places.

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// the sum over a wavefront, in all lanes: 16 lanes by data-parallel moves, the four rows of 16 through scalar registers
__device__ __forceinline__ float wave_total(float v) {
    v = dpp_add<0xb1>(v);
    v = dpp_add<0x4e>(v);
    v = dpp_add<0x141>(v);
    v = dpp_add<0x140>(v);
    auto lane = [&](int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i)); };
    return (lane(0) + lane(16)) + (lane(32) + lane(48));
}
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float (*slots)[TEAM / kWave], int& parity) {
    v = wave_total(v);
    if constexpr (TEAM > kWave) {
        float* const slot = slots[parity];
        parity ^= 1;
        if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TEAM / kWave; ++w) v += slot[w];
    }
    return v;
}

// Sixteen bytes of a row as they are in memory. They stay that way in the registers and are widened where they are used: as an array of
// 16-bit elements the compiler would hold each of them in a register of its own.
typedef __attribute__((ext_vector_type(4))) uint32_t Raw;

template <typename T>
struct Wide;
template <>
struct Wide<float> {
    static constexpr int N = 4;
    static constexpr uint32_t kOnes = 0x3f800000u;
    static __device__ __forceinline__ float up(const Raw& r, int e) { return __uint_as_float(r[e]); }
    static __device__ __forceinline__ Raw down(const float (&f)[N]) {
        return Raw{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
};
template <>
struct Wide<bf16_t> {
    static constexpr int N = 8;
    static constexpr uint32_t kOnes = 0x3f803f80u;
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    static __device__ __forceinline__ float up(const Raw& r, int e) {
        return __uint_as_float(e & 1 ? r[e / 2] & 0xffff0000u : r[e / 2] << 16);
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    }
    static __device__ __forceinline__ Raw down(const float (&f)[N]) {
        return Raw{pair(f[0], f[1]), pair(f[2], f[3]), pair(f[4], f[5]), pair(f[6], f[7])};
    }
};
template <>
struct Wide<f16_t> {
    static constexpr int N = 8;
    static constexpr uint32_t kOnes = 0x3c003c00u;
    typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
    static __device__ __forceinline__ float up(const Raw& r, int e) {
        const uint32_t two = r[e / 2];  // (a bit cast of the vector's element itself takes the vector's first one)
        return (float)__builtin_bit_cast(f16x2, two)[e & 1];
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) { return __builtin_bit_cast(uint32_t, (f16x2{(_Float16)a, (_Float16)b})); }
    static __device__ __forceinline__ Raw down(const float (&f)[N]) {
        return Raw{pair(f[0], f[1]), pair(f[2], f[3]), pair(f[4], f[5]), pair(f[6], f[7])};
    }
};

constexpr int kStream = 2;                // cache policy: non-temporal
constexpr uint32_t kNowhere = 0x7fffffffu;  // an offset past every buffer

// `bytes` at p; nothing where p is NULL. p and bytes are the same in all lanes.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, p ? (int)bytes : 0, 0x00020000);
}
template <bool ELEM, int TEAM, int VPT, int POLICY>
__device__ __forceinline__ void load_row(Raw (&to)[VPT], __amdgpu_buffer_rsrc_t row, int tid) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int at = (tid + i * TEAM) * 16;
        if constexpr (ELEM) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t low = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(row, at + 4 * j, 0, 0);
                to[i][j] = low | (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(row, at + 4 * j + 2, 0, 0) << 16;
            }
        } else {
            to[i] = __builtin_amdgcn_raw_buffer_load_b128(row, at, 0, POLICY);
        }
    }
}
template <bool ELEM, typename T>
__device__ __forceinline__ void store_row(__amdgpu_buffer_rsrc_t row, int v, const float (&f)[Wide<T>::N]) {
    const Raw r = Wide<T>::down(f);
    if constexpr (ELEM) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t two = r[j];
            __builtin_amdgcn_raw_buffer_store_b16((uint16_t)two, row, v * 16 + 4 * j, 0, 0);
            __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(two >> 16), row, v * 16 + 4 * j + 2, 0, 0);
        }
    } else {
        __builtin_amdgcn_raw_buffer_store_b128(r, row, v * 16, 0, kStream);
    }
}
__device__ __forceinline__ float load_float(__amdgpu_buffer_rsrc_t b, uint32_t offset) {
    return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, (int)offset, 0, 0));
}
__device__ __forceinline__ void store_float(__amdgpu_buffer_rsrc_t b, uint32_t offset, float v) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), b, (int)offset, 0, 0);
}
template <typename T>
__device__ __forceinline__ float load_element(__amdgpu_buffer_rsrc_t b) {
    if constexpr (sizeof(T) == 4) return load_float(b, 0);
    else return Num<T>::up(__builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(b, 0, 0, 0)));
}
template <typename T>
__device__ __forceinline__ void store_element(__amdgpu_buffer_rsrc_t b, uint32_t offset, float v) {
    if constexpr (sizeof(T) == 4) store_float(b, offset, v);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, Num<T>::down(v)), b, (int)offset, 0, 0);
}

// a thread's share of a weight, kept over all rows: ones where there is none
template <bool ELEM, typename T, int TEAM, int VPT>
__device__ __forceinline__ void load_weight(Raw (&to)[VPT], const T* p, uint32_t bytes, int tid) {
    load_row<ELEM, TEAM, VPT, 0>(to, buffer_of(p, bytes), tid);
    if (!p) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) to[i] = Wide<T>::kOnes;
    }
}
// Keeps the compiler from widening once and holding the wide values over a barrier
template <int VPT>
__device__ __forceinline__ void stay_packed(Raw (&a)[VPT]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) asm volatile("" : "+v"(a[i]));
}

// index of a team, the same in all of its lanes and known to be
template <int TEAM>
__device__ __forceinline__ int64_t team_index() {
    if constexpr (teams_of(TEAM) == 1) return blockIdx.x;
    else return (int64_t)blockIdx.x * teams_of(TEAM) + __builtin_amdgcn_readfirstlane((int)(threadIdx.x / TEAM));
}

// HBM-bound, each tensor touched once: bf16 [16384, 4096] 89 us, 6.0 TB/s (86 to 96 in a training step), [8188, 2880] with a full gate 41 us, 5.7,
// [4096, 16384] 90 us, 6.0, [32768, 512] 26 us, 5.2; fp32 [16384, 4096] 195 us, 5.5; bf16 [16384, 1031] element by element 106 us, 1.3.
template <typename T, bool ELEM, int TEAM, int VPT, Mode MODE>
__global__ __launch_bounds__(TEAM * teams_of(TEAM)) void sandwich_fwd_kernel(const FwdArgs<T> k) {
    constexpr int N = Wide<T>::N;
    constexpr bool kVector = MODE == kFull || MODE == kGroup;
    __shared__ float s_red[2][TEAM / kWave];
    int parity = 0;
    const int tid = threadIdx.x % TEAM;
    const int64_t H = k.s.H, step = (int64_t)gridDim.x * teams_of(TEAM);
    const uint32_t bytes = (uint32_t)(H * (int64_t)sizeof(T)), first_lane = tid == 0 ? 0u : kNowhere;
    Raw wp[VPT], w[VPT];
    load_weight<ELEM, T, TEAM, VPT>(wp, k.post_weight, bytes, tid);
    load_weight<ELEM, T, TEAM, VPT>(w, k.weight, bytes, tid);
    struct Row {
        Raw x[VPT], r[VPT], gate[VPT];
        float scalar;
    } now, next;
    auto fetch = [&](Row& to, int64_t row) {
        const uint32_t n = row < k.s.B ? bytes : 0u;
        load_row<ELEM, TEAM, VPT, kStream>(to.x, buffer_of(k.x + row * H, n), tid);
        load_row<ELEM, TEAM, VPT, kStream>(to.r, buffer_of(k.residual + row * H, n), tid);
        if constexpr (MODE == kFull) load_row<ELEM, TEAM, VPT, kStream>(to.gate, buffer_of(k.gate + row * H, n), tid);
        if constexpr (MODE == kGroup) load_row<ELEM, TEAM, VPT, 0>(to.gate, buffer_of(k.gate + gate_row(k.s, row) * H, n), tid);
        if constexpr (MODE == kScalar) to.scalar = load_element<T>(buffer_of(k.gate + gate_row(k.s, row), n ? (uint32_t)sizeof(T) : 0u));
    };
    int64_t row = team_index<TEAM>();
    fetch(now, row);
    for (; row < k.s.B; row += step) {
        const int64_t base = row * H;
        fetch(next, row + step);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float v = Wide<T>::up(now.x[i], e);
                ss += v * v;
            }
        const float inv_x = inverse_rms(team_sum<TEAM>(ss, s_red, parity), k.inv_H, k.eps);
        const float a = MODE == kScalar ? k.a * now.scalar : k.a;
        const __amdgpu_buffer_rsrc_t to_stream = buffer_of(k.stream + base, bytes), to_out = buffer_of(k.out + base, bytes);
        float f[VPT][N];
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int v = tid + i * TEAM;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float n = Wide<T>::up(now.x[i], e) * inv_x * Wide<T>::up(wp[i], e);
                if constexpr (kVector) n *= Wide<T>::up(now.gate[i], e);
                f[i][e] = Wide<T>::up(now.r[i], e) + a * n;
                ss += f[i][e] * f[i][e];
            }
            store_row<ELEM, T>(to_stream, v, f[i]);
        }
        const float inv_r = inverse_rms(team_sum<TEAM>(ss, s_red, parity), k.inv_H, k.eps);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float o[N];
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = f[i][e] * inv_r * Wide<T>::up(w[i], e);
            store_row<ELEM, T>(to_out, tid + i * TEAM, o);
        }
        store_float(buffer_of(k.stats ? k.stats + row : nullptr, 4), first_lane, inv_x);
        store_float(buffer_of(k.stats ? k.stats + k.s.B + row : nullptr, 4), first_lane, inv_r);
        now = next;
    }
}

// HBM-bound as well; with the sums over rows, bf16 [16384, 4096] 135 us, 6.0 TB/s, [8188, 2880] with a full gate 71 us, 5.3, [4096, 16384] 160 us,
// 5.0 (rows of more than 1024 vectors have no next row on the way and form r^ three times), [32768, 512] 41 us, 4.9; fp32 [16384, 4096] 274 us,
// 5.9; bf16 [16384, 1031] element by element 159 us, 1.3.
template <typename T, bool ELEM, int TEAM, int VPT, Mode MODE>
__global__ __launch_bounds__(TEAM * teams_of(TEAM)) void sandwich_bwd_kernel(const BwdArgs<T> k) {
    constexpr int N = Wide<T>::N, kTeams = teams_of(TEAM);
    constexpr bool kAhead = TEAM * VPT <= 1024;  // (two vectors for each of 1024 threads leave no registers for a second row)
    constexpr bool kKeep = kAhead;  // (nor for what is formed on the way, which they form again)
    constexpr bool kVector = MODE == kFull || MODE == kGroup || MODE == kChannel;
    __shared__ float s_red[2][TEAM / kWave];
    int parity = 0;
    const int tid = threadIdx.x % TEAM;
    const int64_t H = k.s.H, worker = team_index<TEAM>();
    const uint32_t bytes = (uint32_t)(H * (int64_t)sizeof(T)), first_lane = tid == 0 ? 0u : kNowhere;
    Raw wp[VPT], w[VPT], channel[VPT];
    load_weight<ELEM, T, TEAM, VPT>(wp, k.post_weight, bytes, tid);
    load_weight<ELEM, T, TEAM, VPT>(w, k.weight, bytes, tid);
    if constexpr (MODE == kChannel) load_row<ELEM, TEAM, VPT, 0>(channel, buffer_of(k.gate, bytes), tid);
    float sw[VPT][N], swp[VPT][N], sg[VPT][N];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) sw[i][e] = swp[i][e] = sg[i][e] = 0.f;

    struct Row {
        Raw x[VPT], r[VPT], dy[VPT], dr[VPT], gate[VPT];
        float inv_x, inv_r, scalar;
    } now, next;
    auto fetch = [&](Row& to, int64_t row, bool in) {
        const int64_t base = row * H;
        const uint32_t n = in ? bytes : 0u, one = in ? 4u : 0u;
        load_row<ELEM, TEAM, VPT, kStream>(to.x, buffer_of(k.x + base, n), tid);
        load_row<ELEM, TEAM, VPT, kStream>(to.r, buffer_of(k.residual + base, n), tid);
        load_row<ELEM, TEAM, VPT, kStream>(to.dy, buffer_of(k.d_out ? k.d_out + base : nullptr, n), tid);
        load_row<ELEM, TEAM, VPT, kStream>(to.dr, buffer_of(k.d_stream ? k.d_stream + base : nullptr, n), tid);
        if constexpr (MODE == kFull) load_row<ELEM, TEAM, VPT, kStream>(to.gate, buffer_of(k.gate + base, n), tid);
        if constexpr (MODE == kGroup) load_row<ELEM, TEAM, VPT, 0>(to.gate, buffer_of(k.gate + gate_row(k.s, row) * H, n), tid);
        if constexpr (MODE == kScalar) to.scalar = load_element<T>(buffer_of(k.gate + gate_row(k.s, row), in ? (uint32_t)sizeof(T) : 0u));
        to.inv_x = load_float(buffer_of(k.stats + row, one), 0);
        to.inv_r = load_float(buffer_of(k.stats + k.s.B + row, one), 0);
    };
    // the rows of a group `parts` apart, then the next group: rows in flight at the same time are neighbours in memory
    const int64_t part = worker % k.p.parts, groups = k.p.workers / k.p.parts;
    int64_t group = worker / k.p.parts, place = part;
    bool more = worker < k.p.workers;
    if constexpr (kAhead) fetch(now, group * k.p.rows + place, more);
    while (more) {
        const int64_t row = group * k.p.rows + place, base = row * H;
        int64_t next_group = group, next_place = place + k.p.parts;
        if (next_place >= k.p.rows) {
            next_place = part;
            next_group += groups;
        }
        more = next_group < k.p.groups;
        if constexpr (kAhead) fetch(next, next_group * k.p.rows + next_place, more);
        else fetch(now, row, true);

        auto gate = [&](int i, int e) {
            if constexpr (MODE == kChannel) return Wide<T>::up(channel[i], e);
            else return Wide<T>::up(now.gate[i], e);
        };
        const float a = MODE == kScalar ? k.a * now.scalar : k.a;
        // r^, from the stream as it was before its rounding
        const float x_share = a * now.inv_x * now.inv_r;
        auto form = [&](int i, int e) {
            float n = Wide<T>::up(now.x[i], e) * Wide<T>::up(wp[i], e);
            if constexpr (kVector) n *= gate(i, e);
            return Wide<T>::up(now.r[i], e) * now.inv_r + n * x_share;
        };
        float kept[VPT][N];  // a number per element over the barriers: first r^, then dr
        if constexpr (kKeep) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) kept[i][e] = form(i, e);
        }
        auto normed = [&](int i, int e) {
            if constexpr (kKeep) return kept[i][e];
            else return form(i, e);
        };
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) dot += Wide<T>::up(now.dy[i], e) * Wide<T>::up(w[i], e) * normed(i, e);
        const float c_r = team_sum<TEAM>(dot, s_red, parity) * k.inv_H;
        auto d_stream = [&](int i, int e, float dy, float rh) {
            return Wide<T>::up(now.dr[i], e) + now.inv_r * (dy * Wide<T>::up(w[i], e) - rh * c_r);
        };
        auto stay = [&](bool formed) {
            stay_packed(now.x);
            if constexpr (!kKeep) stay_packed(now.r);
            if (!kKeep || !formed) {
                stay_packed(now.dy);
                stay_packed(now.dr);
                stay_packed(w);
            }
            stay_packed(wp);
            if constexpr (MODE == kChannel) stay_packed(channel);
            else if constexpr (kVector) stay_packed(now.gate);
        };
        stay(false);
        const __amdgpu_buffer_rsrc_t to_residual = buffer_of(k.d_residual + base, bytes), to_x = buffer_of(k.dx + base, bytes);
        dot = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float o[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float dy = Wide<T>::up(now.dy[i], e), rh = normed(i, e), dr = d_stream(i, e, dy, rh);
                sw[i][e] += dy * rh;
                float u = dr * Wide<T>::up(wp[i], e);
                if constexpr (kVector) u *= gate(i, e);
                dot += u * Wide<T>::up(now.x[i], e);
                o[e] = dr;
                if constexpr (kKeep) kept[i][e] = dr;
            }
            store_row<ELEM, T>(to_residual, tid + i * TEAM, o);
        }
        dot = team_sum<TEAM>(dot, s_red, parity) * now.inv_x;
        if constexpr (MODE == kScalar) {
            const bool own = k.d_gate && k.s.R == 1;  // the row's number is the gate's gradient, or one of those it sums
            store_element<T>(buffer_of(own ? k.d_gate + row : nullptr, sizeof(T)), first_lane, k.a * dot);
            store_float(buffer_of(own || !k.d_gate ? nullptr : k.part.rows + row, 4), first_lane, k.a * dot);
        }
        const float c_x = a * dot * k.inv_H;
        stay(true);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float o[N], og[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float xh = Wide<T>::up(now.x[i], e) * now.inv_x, p = Wide<T>::up(wp[i], e);
                float dr;
                if constexpr (kKeep) dr = kept[i][e];
                else dr = d_stream(i, e, Wide<T>::up(now.dy[i], e), normed(i, e));
                const float dz = a * dr;  // (kScalar: a with the row's gate in it)
                float gated = dz;
                if constexpr (kVector) gated *= gate(i, e);
                o[e] = now.inv_x * (gated * p - xh * c_x);
                og[e] = dz * p * xh;
                swp[i][e] += (MODE == kChannel ? dz : gated) * xh;
                if constexpr (MODE == kGroup) sg[i][e] += dz * xh;
            }
            store_row<ELEM, T>(to_x, tid + i * TEAM, o);
            if constexpr (MODE == kFull) store_row<ELEM, T>(buffer_of(k.d_gate ? k.d_gate + base : nullptr, bytes), tid + i * TEAM, og);
        }
        if constexpr (MODE == kGroup)
            if (!more || next_group != group) {  // the group's sum is whole here, or this team's part of it
                const __amdgpu_buffer_rsrc_t to_gate = buffer_of(k.d_gate && k.p.parts == 1 ? k.d_gate + group * H : nullptr, bytes);
                const __amdgpu_buffer_rsrc_t to_part =
                    buffer_of(k.d_gate && k.p.parts > 1 ? k.part.gate + worker * H : nullptr, (uint32_t)(H * 4));
#pragma unroll
                for (int i = 0; i < VPT; ++i) {
                    const int v = tid + i * TEAM;
                    float o[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        o[e] = sg[i][e] * Wide<T>::up(wp[i], e);
                        store_float(to_part, (uint32_t)(v * N + e) * 4, sg[i][e]);
                        sg[i][e] = 0.f;
                    }
                    store_row<ELEM, T>(to_gate, v, o);
                }
            }
        if constexpr (kAhead) now = next;
        group = next_group;
        place = next_place;
    }
    // the partial sums of a workgroup's teams together, in order
    const __amdgpu_buffer_rsrc_t to_w = buffer_of(k.sums_w ? k.part.w + (int64_t)blockIdx.x * H : nullptr, (uint32_t)(H * 4));
    const __amdgpu_buffer_rsrc_t to_wp = buffer_of(k.sums_wp ? k.part.wp + (int64_t)blockIdx.x * H : nullptr, (uint32_t)(H * 4));
    if constexpr (kTeams == 1) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                auto four = [&](const float (&f)[N]) {
                    return Raw{__float_as_uint(f[e]), __float_as_uint(f[e + 1]), __float_as_uint(f[e + 2]), __float_as_uint(f[e + 3])};
                };
                __builtin_amdgcn_raw_buffer_store_b128(four(sw[i]), to_w, ((tid + i * TEAM) * N + e) * 4, 0, 0);
                __builtin_amdgcn_raw_buffer_store_b128(four(swp[i]), to_wp, ((tid + i * TEAM) * N + e) * 4, 0, 0);
            }
    } else {
        __shared__ float s_sum[kTeams][TEAM * VPT * N];
        auto join = [&](const float (&f)[VPT][N], __amdgpu_buffer_rsrc_t to) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) s_sum[threadIdx.x / TEAM][(tid + i * TEAM) * N + e] = f[i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < TEAM * VPT * N; c += TEAM * kTeams) {
                float t = 0.f;
#pragma unroll
                for (int j = 0; j < kTeams; ++j) t += s_sum[j][c];
                store_float(to, (uint32_t)c * 4, t);
            }
        };
        join(sw, to_w);
        join(swp, to_wp);
    }
}

// ---- sums over rows -----------------------------------------------------------------------------------------------------------

template <typename T>
struct ReduceArgs {
    Partial part;
    const T *post_weight, *gate;
    T *d_weight, *d_post_weight, *d_gate;
    Shape s;
    Split p;
};

// A workgroup owns 32 columns; its 32 groups of 32 threads each add every 32nd row in 64 bits, and the 32 results are added in order.
// blockIdx.y: 0 dw, 1 dw_post (and with kChannel dgate, which is the same sum), 2 .. the rows of dgate (kGroup).
constexpr int kReduceThreads = 1024, kReduceCols = 32, kReduceGroups = kReduceThreads / kReduceCols;
template <typename T>
__global__ __launch_bounds__(kReduceThreads) void sandwich_reduce_kernel(const ReduceArgs<T> k) {
    __shared__ double s_acc[kReduceGroups][kReduceCols];
    const int col = threadIdx.x % kReduceCols, group = threadIdx.x / kReduceCols;
    const int64_t H = k.s.H, h = (int64_t)blockIdx.x * kReduceCols + col;
    const int what = (int)blockIdx.y;
    const bool channel = k.s.mode == kChannel;
    if (what == 0 ? !k.d_weight : what == 1 ? !(k.d_post_weight || (channel && k.d_gate)) : !k.d_gate) return;
    const float* p = what == 0 ? k.part.w : what == 1 ? k.part.wp : k.part.gate + (int64_t)(what - 2) * k.p.parts * H;
    const int64_t rows = what < 2 ? k.p.sums : k.p.parts;
    double acc = 0.0;
    if (h < H) {
        int64_t g = group;
        for (; g + 3 * kReduceGroups < rows; g += 4 * kReduceGroups) {
            const float a0 = p[g * H + h], a1 = p[(g + kReduceGroups) * H + h];
            const float a2 = p[(g + 2 * kReduceGroups) * H + h], a3 = p[(g + 3 * kReduceGroups) * H + h];
            acc += (double)a0;
            acc += (double)a1;
            acc += (double)a2;
            acc += (double)a3;
        }
        for (; g < rows; g += kReduceGroups) acc += (double)p[g * H + h];
    }
    s_acc[group][col] = acc;
    __syncthreads();
    if (group != 0 || h >= H) return;
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < kReduceGroups; ++i) total += s_acc[i][col];
    if (what == 0) k.d_weight[h] = Num<T>::down((float)total);
    else if (what == 1) {
        if (k.d_post_weight) k.d_post_weight[h] = Num<T>::down((float)(total * (channel ? at(k.gate, h) : 1.0f)));
        if (channel && k.d_gate) k.d_gate[h] = Num<T>::down((float)(total * at(k.post_weight, h)));
    } else k.d_gate[(int64_t)(what - 2) * H + h] = Num<T>::down((float)(total * at(k.post_weight, h)));
}

// the rows' numbers to those of a gate [G, 1]
template <typename T>
__global__ __launch_bounds__(kThreads) void sandwich_reduce_scalar_kernel(const float* __restrict__ rows, int64_t G, int64_t R, T* __restrict__ d_gate) {
    __shared__ double s_acc[kThreads];
    for (int64_t g = blockIdx.x; g < G; g += gridDim.x) {
        double acc = 0.0;
        for (int64_t i = threadIdx.x; i < R; i += kThreads) acc += (double)rows[g * R + i];
        __syncthreads();
        s_acc[threadIdx.x] = acc;
        __syncthreads();
        for (int d = kThreads / 2; d > 0; d >>= 1) {
            if ((int)threadIdx.x < d) s_acc[threadIdx.x] += s_acc[threadIdx.x + d];
            __syncthreads();
        }
        if (threadIdx.x == 0) d_gate[g] = Num<T>::down((float)s_acc[0]);
    }
}

// ---- launch -------------------------------------------------------------------------------------------------------------------

template <int TEAM, int VPT, bool ELEM = false>
struct Team {
    static constexpr int team = TEAM, vpt = VPT;
    static constexpr bool elem = ELEM;
};
// calls `launch` with the team of a row of nvec vectors, the last of which may not be full, as a type; false: no team holds it
template <typename T, typename F>
bool with_team(int64_t nvec, bool dwords, F launch) {
    if (nvec > 2048) return false;
    if constexpr (sizeof(T) == 2)
        if (!dwords) {
            if (nvec <= 128) launch(Team<64, 2, true>());
            else if (nvec <= 256) launch(Team<256, 1, true>());
            else if (nvec <= 512) launch(Team<512, 1, true>());
            else if (nvec <= 1024) launch(Team<1024, 1, true>());
            else launch(Team<1024, 2, true>());
            return true;
        }
    if (nvec <= 64) launch(Team<64, 1>());
    else if (nvec <= 128) launch(Team<64, 2>());
    else if (nvec <= 256) launch(Team<256, 1>());
    else if (nvec <= 384) launch(Team<384, 1>());
    else if (nvec <= 512) launch(Team<512, 1>());
    else if (nvec <= 768) launch(Team<768, 1>());
    else if (nvec <= 1024) launch(Team<1024, 1>());
    else launch(Team<1024, 2>());
    return true;
}
template <typename T>
int64_t vectors_of(int64_t H) {
    return (H * (int64_t)sizeof(T) + 15) / 16;
}
// whether all rows start on a dword boundary
template <typename T>
bool dwords_of(int64_t H, std::initializer_list<const void*> pointers) {
    bool fine = H * (int64_t)sizeof(T) % 4 == 0;
    for (const void* p : pointers) fine = fine && ((uintptr_t)p & 3u) == 0;
    return fine;
}
template <Mode MODE>
using As = std::integral_constant<Mode, MODE>;

template <typename T>
int launch_fwd(const FwdArgs<T>& k, hipStream_t st) {
    const int64_t cus = num_compute_units() > 0 ? num_compute_units() : 256;
    const bool dwords = dwords_of<T>(k.s.H, {k.x, k.residual, k.post_weight, k.weight, k.s.mode == kScalar ? nullptr : k.gate, k.out, k.stream});
    const bool held = with_team<T>(vectors_of<T>(k.s.H), dwords, [&](auto t) {
        constexpr int TEAM = decltype(t)::team, VPT = decltype(t)::vpt;
        constexpr int kTeams = teams_of(TEAM);
        const int64_t want = (k.s.B + kTeams - 1) / kTeams, most = cus * (kFwdThreadsPerCU / (TEAM * kTeams));
        auto launch = [&](auto mode) {
            hipLaunchKernelGGL((sandwich_fwd_kernel<T, decltype(t)::elem, TEAM, VPT, decltype(mode)::value>), dim3((uint32_t)(want < most ? want : most)),
                               dim3(TEAM * kTeams), 0, st, k);
        };
        switch (k.s.mode) {
            case kNoGate: launch(As<kNoGate>()); break;
            case kFull: launch(As<kFull>()); break;
            case kScalar: launch(As<kScalar>()); break;
            default: launch(As<kGroup>()); break;
        }
    });
    const int64_t most = cus * 16;
    if (!held)
        hipLaunchKernelGGL(sandwich_fwd_generic_kernel<T>, dim3((uint32_t)(k.s.B < most ? k.s.B : most)), dim3(kThreads), 0, st, k);
    return launch_status("sandwich_rmsnorm_fwd");
}

template <typename T>
int launch_bwd(BwdArgs<T> k, T* d_weight, T* d_post_weight, void* workspace, hipStream_t st) {
    k.p = split_of(k.s, kThreads, 1);  // of the element-wise kernel
    k.part = partial_of(workspace, k.s, k.p);
    const bool dwords = dwords_of<T>(k.s.H, {k.x, k.residual, k.post_weight, k.weight, k.s.mode == kScalar ? nullptr : k.gate, k.d_out, k.d_stream, k.dx,
                                             k.d_residual, k.s.mode == kScalar ? nullptr : k.d_gate});
    const bool held = with_team<T>(vectors_of<T>(k.s.H), dwords, [&](auto t) {
        constexpr int TEAM = decltype(t)::team, VPT = decltype(t)::vpt;
        k.p = split_of(k.s, TEAM, teams_of(TEAM));
        k.part = partial_of(workspace, k.s, k.p);
        auto launch = [&](auto mode) {
            hipLaunchKernelGGL((sandwich_bwd_kernel<T, decltype(t)::elem, TEAM, VPT, decltype(mode)::value>), dim3((uint32_t)k.p.sums), dim3(TEAM * teams_of(TEAM)), 0,
                               st, k);
        };
        switch (k.s.mode) {
            case kNoGate: launch(As<kNoGate>()); break;
            case kFull: launch(As<kFull>()); break;
            case kChannel: launch(As<kChannel>()); break;
            case kScalar: launch(As<kScalar>()); break;
            default: launch(As<kGroup>()); break;
        }
    });
    if (!held) hipLaunchKernelGGL(sandwich_bwd_generic_kernel<T>, dim3((uint32_t)k.p.workers), dim3(kThreads), 0, st, k);
    int rc = launch_status("sandwich_rmsnorm_bwd");
    if (rc) return rc;
    const ReduceArgs<T> r{k.part, k.post_weight, k.gate, d_weight, d_post_weight, k.d_gate, k.s, k.p};
    const int64_t groups = k.s.mode == kGroup && k.d_gate && k.p.parts > 1 ? k.p.groups : 0;
    if (d_weight || d_post_weight || (k.s.mode == kChannel && k.d_gate) || groups) {
        hipLaunchKernelGGL(sandwich_reduce_kernel<T>, dim3((uint32_t)((k.s.H + kReduceCols - 1) / kReduceCols), (uint32_t)(2 + groups)),
                           dim3(kReduceThreads), 0, st, r);
        rc = launch_status("sandwich_rmsnorm_bwd (sums)");
        if (rc) return rc;
    }
    if (k.s.mode == kScalar && k.d_gate && k.s.R > 1) {
        const int64_t G = k.s.B / k.s.R;
        hipLaunchKernelGGL(sandwich_reduce_scalar_kernel<T>, dim3((uint32_t)(G < 4096 ? G : 4096)), dim3(kThreads), 0, st, k.part.rows, G, k.s.R, k.d_gate);
        return launch_status("sandwich_rmsnorm_bwd (gate)");
    }
    return FMA_OK;
}

int check(const char* what, int64_t B, int64_t H, const void* gate, int64_t gate_rows, int64_t gate_width, int dtype) {
    FMA_REQUIRE(dtype_bytes(dtype) != 0, FMA_ERR_BAD_DTYPE, "%s: unknown dtype code %d", what, dtype);
    FMA_REQUIRE(B >= 0 && B <= 0x7fffffffll, FMA_ERR_BAD_SIZE, "%s: bad row count %lld", what, (long long)B);
    FMA_REQUIRE(H >= 1 && H <= FMA_MAX_NORM_HIDDEN, FMA_ERR_BAD_SIZE, "%s: H must be in [1, %d] (got %lld)", what, FMA_MAX_NORM_HIDDEN,
                (long long)H);
    if (gate) {
        FMA_REQUIRE(gate_width == H || gate_width == 1, FMA_ERR_BAD_SIZE, "%s: a gate has 1 or %lld columns (got %lld)", what, (long long)H,
                    (long long)gate_width);
        FMA_REQUIRE(gate_rows >= 1 && (B == 0 || (gate_rows <= B && B % gate_rows == 0)), FMA_ERR_BAD_SIZE,
                    "%s: the gate's %lld rows do not divide %lld", what, (long long)gate_rows, (long long)B);
    }
    return FMA_OK;
}

bool aligned_to_elements(std::initializer_list<const void*> pointers, int dtype) {
    for (const void* p : pointers)
        if ((uintptr_t)p & (uintptr_t)(dtype_bytes(dtype) - 1)) return false;
    return true;
}

template <typename T>
int forward(const void* x, const void* residual, const void* post_weight, const void* weight, const void* gate, void* out, void* stream,
            float* stats, const Shape& s, float eps, float a, hipStream_t st) {
    const FwdArgs<T> k{(const T*)x, (const T*)residual, (const T*)post_weight, (const T*)weight, (const T*)gate, (T*)out, (T*)stream, stats, s,
                       1.0f / (float)s.H, eps, a};
    return launch_fwd(k, st);
}

template <typename T>
int backward(const void* x, const void* residual, const void* post_weight, const void* weight, const void* gate, const void* d_out,
             const void* d_stream, const float* stats, void* dx, void* d_residual, void* d_gate, void* d_post_weight, void* d_weight,
             const Shape& s, float a, void* workspace, hipStream_t st) {
    const BwdArgs<T> k{(const T*)x, (const T*)residual, (const T*)post_weight, (const T*)weight, (const T*)gate, (const T*)d_out, (const T*)d_stream,
                       stats, (T*)dx, (T*)d_residual, (T*)d_gate, Partial{}, s, Split{}, 1.0f / (float)s.H, a, d_weight != nullptr,
                       d_post_weight != nullptr || (s.mode == kChannel && d_gate)};
    return launch_bwd<T>(k, (T*)d_weight, (T*)d_post_weight, workspace, st);
}

}  // namespace
}  // namespace fmahip

extern "C" {

int fma_sandwich_rmsnorm_fwd(const void* x, const void* residual, const void* post_weight, const void* weight, const void* gate,
                             int64_t gate_rows, int64_t gate_width, void* out, void* stream_out, float* stats, int64_t B, int64_t H, float eps,
                             float multiplier, int dtype, void* stream) {
    using namespace fmahip;
    const int rc = check("sandwich_rmsnorm_fwd", B, H, gate, gate_rows, gate_width, dtype);
    if (rc || B == 0) return rc;
    FMA_REQUIRE(x && residual && out && stream_out, FMA_ERR_NULL_POINTER, "sandwich_rmsnorm_fwd: NULL pointer");
    FMA_REQUIRE(aligned_to_elements({x, residual, post_weight, weight, gate, out, stream_out}, dtype), FMA_ERR_MISALIGNED,
                "sandwich_rmsnorm_fwd: tensors must be aligned to their elements");
    const Shape s = shape_of(B, H, gate ? gate_rows : 0, gate_width);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case FMA_F32: return forward<float>(x, residual, post_weight, weight, gate, out, stream_out, stats, s, eps, multiplier, st);
        case FMA_F16: return forward<f16_t>(x, residual, post_weight, weight, gate, out, stream_out, stats, s, eps, multiplier, st);
        default: return forward<bf16_t>(x, residual, post_weight, weight, gate, out, stream_out, stats, s, eps, multiplier, st);
    }
}

int64_t fma_sandwich_rmsnorm_bwd_workspace_bytes(int64_t B, int64_t H, int64_t gate_rows, int64_t gate_width) {
    if (B <= 0 || H <= 0 || gate_rows < 0 || gate_rows > B) return 0;
    return fmahip::workspace_bytes_of(fmahip::shape_of(B, H, gate_rows, gate_width));
}

int fma_sandwich_rmsnorm_bwd(const void* x, const void* residual, const void* post_weight, const void* weight, const void* gate,
                             int64_t gate_rows, int64_t gate_width, const void* out_grad, const void* stream_grad, const float* stats,
                             void* x_grad, void* residual_grad, void* gate_grad, void* post_weight_grad, void* weight_grad, int64_t B, int64_t H,
                             float multiplier, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
    using namespace fmahip;
    const int rc = check("sandwich_rmsnorm_bwd", B, H, gate, gate_rows, gate_width, dtype);
    if (rc) return rc;
    FMA_REQUIRE((gate || !gate_grad) && (post_weight || !post_weight_grad) && (weight || !weight_grad), FMA_ERR_NULL_POINTER,
                "sandwich_rmsnorm_bwd: a gradient without its input");
    FMA_REQUIRE(B > 0, FMA_ERR_BAD_SIZE, "sandwich_rmsnorm_bwd: no rows");
    FMA_REQUIRE(x && residual && stats && x_grad && residual_grad, FMA_ERR_NULL_POINTER, "sandwich_rmsnorm_bwd: NULL pointer");
    FMA_REQUIRE(aligned_to_elements({x, residual, post_weight, weight, gate, out_grad, stream_grad, x_grad, residual_grad, gate_grad,
                                     post_weight_grad, weight_grad}, dtype),
                FMA_ERR_MISALIGNED, "sandwich_rmsnorm_bwd: tensors must be aligned to their elements");
    const Shape s = shape_of(B, H, gate ? gate_rows : 0, gate_width);
    const int64_t need = workspace_bytes_of(s);
    FMA_REQUIRE(workspace, FMA_ERR_NULL_POINTER, "sandwich_rmsnorm_bwd: NULL workspace");
    FMA_REQUIRE(workspace_bytes >= need, FMA_ERR_WORKSPACE_TOO_SMALL, "sandwich_rmsnorm_bwd: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
    FMA_REQUIRE(((uintptr_t)workspace & 15u) == 0, FMA_ERR_MISALIGNED, "sandwich_rmsnorm_bwd: workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case FMA_F32:
            return backward<float>(x, residual, post_weight, weight, gate, out_grad, stream_grad, stats, x_grad, residual_grad, gate_grad,
                                   post_weight_grad, weight_grad, s, multiplier, workspace, st);
        case FMA_F16:
            return backward<f16_t>(x, residual, post_weight, weight, gate, out_grad, stream_grad, stats, x_grad, residual_grad, gate_grad,
                                   post_weight_grad, weight_grad, s, multiplier, workspace, st);
        default:
            return backward<bf16_t>(x, residual, post_weight, weight, gate, out_grad, stream_grad, stats, x_grad, residual_grad, gate_grad,
                                    post_weight_grad, weight_grad, s, multiplier, workspace, st);
    }
}

}  // extern "C"
