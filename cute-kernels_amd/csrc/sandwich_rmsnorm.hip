// The norm behind a block, its gate and residual scale, the residual stream and the norm before the next block, forward and backward:
//
//   n   = x inv_x w_post            inv_x = 1 / sqrt(mean(x^2) + eps)
//   r   = residual + a gate n       (stored rounded; a: the residual scale)
//   out = r inv_r w                 inv_r = 1 / sqrt(mean(r^2) + eps), from the unrounded r
//
// with x^ = x inv_x, r^ = r inv_r (from the stored r), g = dout w:
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
constexpr int kBwdPerCU = 2;

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

// The workgroups of the backward pass: `parts` for each of `groups` of neighbouring rows (one group unless the gate has several rows that
// serve several rows each), or, with more groups than workgroups are wanted, whole groups for each.
struct Split {
    int64_t groups, rows, parts, workgroups;
};
Split split_of(const Shape& s) {
    const int64_t cus = num_compute_units() > 0 ? num_compute_units() : 256, want = cus * kBwdPerCU;
    Split p{1, s.B, 1, 1};
    if (s.mode == kGroup) {
        p.groups = s.B / s.R;
        p.rows = s.R;
    }
    p.parts = want / p.groups;
    if (p.parts > p.rows) p.parts = p.rows;
    if (p.parts < 1) p.parts = 1;
    p.workgroups = p.parts > 1 || p.groups <= want ? p.groups * p.parts : want;
    return p;
}

// the workspace: partial sums [workgroups, H] for dw, dw_post and (kGroup) dgate, one number per row (kScalar)
struct Partial {
    float *w, *wp, *gate, *rows;
};
Partial partial_of(void* workspace, const Shape& s, const Split& p) {
    const int64_t n = p.workgroups * s.H;
    Partial part;
    part.w = (float*)workspace;
    part.wp = part.w + n;
    part.gate = part.wp + n;
    part.rows = part.wp + n;
    return part;
}
int64_t workspace_bytes_of(const Shape& s) {
    return 4 * (split_of(s).workgroups * s.H * (s.mode == kGroup ? 3 : 2) + (s.mode == kScalar ? s.B : 0));
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
    const T *x, *stream, *post_weight, *weight, *gate, *d_out, *d_stream;
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

// ---- any H, any alignment: element by element -----------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(kThreads) void sandwich_fwd_generic_kernel(const FwdArgs<T> k) {
    __shared__ float s_red[2][kWaves];
    int parity = 0;
    const int64_t H = k.s.H;
    for (int64_t row = blockIdx.x; row < k.s.B; row += gridDim.x) {
        const int64_t base = row * H;
        const T* const gate = k.gate ? k.gate + row / k.s.R * (k.s.mode == kScalar ? 1 : H) : nullptr;
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
            const T* const gate = k.gate ? k.gate + row / k.s.R * (scalar ? 1 : H) : nullptr;
            const float inv_x = k.stats[row], inv_r = k.stats[k.s.B + row];
            float dot = 0.f;
            if (k.d_out)
                for (int64_t h = threadIdx.x; h < H; h += kThreads)
                    dot += Num<T>::up(k.d_out[base + h]) * at(k.weight, h) * Num<T>::up(k.stream[base + h]);
            const float c_r = workgroup_sum(dot, s_red, parity) * inv_r * k.inv_H;
            auto d_stream = [&](int64_t h) {
                float d = k.d_stream ? Num<T>::up(k.d_stream[base + h]) : 0.f;
                if (k.d_out) d += inv_r * (Num<T>::up(k.d_out[base + h]) * at(k.weight, h) - Num<T>::up(k.stream[base + h]) * inv_r * c_r);
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
                if (w) w[h] += k.d_out ? Num<T>::up(k.d_out[base + h]) * (Num<T>::up(k.stream[base + h]) * inv_r) : 0.f;
                if (wp) wp[h] += k.s.mode == kChannel ? dz * x : dz * g * x;
                if (sg) sg[h] += dz * x;
            }
        }
        if (sg && k.p.parts == 1)
            for (int64_t h = threadIdx.x; h < H; h += kThreads) k.d_gate[group * H + h] = Num<T>::down(at(k.post_weight, h) * sg[h]);
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

// A workgroup owns 32 columns; its 8 groups of 32 threads each add every 8th row in 64 bits, and the 8 results are added in order.
// blockIdx.y: 0 dw, 1 dw_post (and with kChannel dgate, which is the same sum), 2 .. the rows of dgate (kGroup).
constexpr int kReduceCols = 32, kReduceGroups = kThreads / kReduceCols;
template <typename T>
__global__ __launch_bounds__(kThreads) void sandwich_reduce_kernel(const ReduceArgs<T> k) {
    __shared__ double s_acc[kReduceGroups][kReduceCols];
    const int col = threadIdx.x % kReduceCols, group = threadIdx.x / kReduceCols;
    const int64_t H = k.s.H, h = (int64_t)blockIdx.x * kReduceCols + col;
    const int what = (int)blockIdx.y;
    const bool channel = k.s.mode == kChannel;
    if (what == 0 ? !k.d_weight : what == 1 ? !(k.d_post_weight || (channel && k.d_gate)) : !k.d_gate) return;
    const float* p = what == 0 ? k.part.w : what == 1 ? k.part.wp : k.part.gate + (int64_t)(what - 2) * k.p.parts * H;
    const int64_t rows = what < 2 ? k.p.workgroups : k.p.parts;
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

template <typename T>
int launch_fwd(const FwdArgs<T>& k, hipStream_t st) {
    const int64_t cus = num_compute_units() > 0 ? num_compute_units() : 256, most = cus * 16;
    const dim3 grid((uint32_t)(k.s.B < most ? k.s.B : most));
    hipLaunchKernelGGL(sandwich_fwd_generic_kernel<T>, grid, dim3(kThreads), 0, st, k);
    return launch_status("sandwich_rmsnorm_fwd");
}

template <typename T>
int launch_bwd(const BwdArgs<T>& k, T* d_weight, T* d_post_weight, hipStream_t st) {
    if (k.s.B > 0) {
        hipLaunchKernelGGL(sandwich_bwd_generic_kernel<T>, dim3((uint32_t)k.p.workgroups), dim3(kThreads), 0, st, k);
        const int rc = launch_status("sandwich_rmsnorm_bwd");
        if (rc) return rc;
    }
    const ReduceArgs<T> r{k.part, k.post_weight, k.gate, d_weight, d_post_weight, k.d_gate, k.s, k.p};
    const int64_t groups = k.s.mode == kGroup && k.d_gate && k.p.parts > 1 ? k.p.groups : 0;
    if (d_weight || d_post_weight || (k.s.mode == kChannel && k.d_gate) || groups) {
        hipLaunchKernelGGL(sandwich_reduce_kernel<T>, dim3((uint32_t)((k.s.H + kReduceCols - 1) / kReduceCols), (uint32_t)(2 + groups)),
                           dim3(kThreads), 0, st, r);
        const int rc = launch_status("sandwich_rmsnorm_bwd (sums)");
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
int backward(const void* x, const void* stream, const void* post_weight, const void* weight, const void* gate, const void* d_out,
             const void* d_stream, const float* stats, void* dx, void* d_residual, void* d_gate, void* d_post_weight, void* d_weight,
             const Shape& s, float a, void* workspace, hipStream_t st) {
    const Split p = split_of(s);
    const BwdArgs<T> k{(const T*)x, (const T*)stream, (const T*)post_weight, (const T*)weight, (const T*)gate, (const T*)d_out, (const T*)d_stream,
                       stats, (T*)dx, (T*)d_residual, (T*)d_gate, partial_of(workspace, s, p), s, p, 1.0f / (float)s.H, a, d_weight != nullptr,
                       d_post_weight != nullptr || (s.mode == kChannel && d_gate)};
    return launch_bwd<T>(k, (T*)d_weight, (T*)d_post_weight, st);
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

int fma_sandwich_rmsnorm_bwd(const void* x, const void* stream_out, const void* post_weight, const void* weight, const void* gate,
                             int64_t gate_rows, int64_t gate_width, const void* out_grad, const void* stream_grad, const float* stats,
                             void* x_grad, void* residual_grad, void* gate_grad, void* post_weight_grad, void* weight_grad, int64_t B, int64_t H,
                             float multiplier, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
    using namespace fmahip;
    const int rc = check("sandwich_rmsnorm_bwd", B, H, gate, gate_rows, gate_width, dtype);
    if (rc) return rc;
    FMA_REQUIRE((gate || !gate_grad) && (post_weight || !post_weight_grad) && (weight || !weight_grad), FMA_ERR_NULL_POINTER,
                "sandwich_rmsnorm_bwd: a gradient without its input");
    FMA_REQUIRE(B > 0, FMA_ERR_BAD_SIZE, "sandwich_rmsnorm_bwd: no rows");
    FMA_REQUIRE(x && stream_out && stats && x_grad && residual_grad, FMA_ERR_NULL_POINTER, "sandwich_rmsnorm_bwd: NULL pointer");
    FMA_REQUIRE(aligned_to_elements({x, stream_out, post_weight, weight, gate, out_grad, stream_grad, x_grad, residual_grad, gate_grad,
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
            return backward<float>(x, stream_out, post_weight, weight, gate, out_grad, stream_grad, stats, x_grad, residual_grad, gate_grad,
                                   post_weight_grad, weight_grad, s, multiplier, workspace, st);
        case FMA_F16:
            return backward<f16_t>(x, stream_out, post_weight, weight, gate, out_grad, stream_grad, stats, x_grad, residual_grad, gate_grad,
                                   post_weight_grad, weight_grad, s, multiplier, workspace, st);
        default:
            return backward<bf16_t>(x, stream_out, post_weight, weight, gate, out_grad, stream_grad, stats, x_grad, residual_grad, gate_grad,
                                    post_weight_grad, weight_grad, s, multiplier, workspace, st);
    }
}

}  // extern "C"
