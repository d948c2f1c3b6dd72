// The norm of many tensors together, and scaling them down to a bound:
//
//   norm = sqrt(sum over all elements of all tensors of g^2)   or   max |g|
//   g   *= min(1, max_norm / (norm + 1e-6))
//
// HBM-bound: one pass reads every element, a second reads and writes it. Squares are added in 64 bits from the first one on: in 32 bits
// a gradient of 2^64 or of 2^-75 would already be lost in its square. Tensors come as a table in the kernel's arguments (no table in
// device memory that a captured graph or a second call would have to share), cut into chunks.
#include "common.h"

#include <stdlib.h>

#include <algorithm>
#include <type_traits>

namespace fmahip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// Elements of a chunk; multiples of every 16-byte vector, so that all chunks of a tensor are aligned alike
constexpr int kNormChunk = 16384, kScaleChunk = 8192;
constexpr int kTable = 160;         // tensors per launch: 3.4 KB of kernel arguments
constexpr int kNormPerCU = 8;       // workgroups per compute unit; the scaling has one for every chunk
constexpr int64_t kMostGrid = 1 << 22;
// Bytes of all tensors from which on they are read and written as a stream (non-temporal), and not left in the caches for the second pass. us of
// norm and scaling, streamed / not: 68 MB 42 / 38, 151 MB 79 / 93, 302 MB 149 / 178, 2.2 GB 1061 / 1202.
constexpr int64_t kStreamBytes = 128ll << 20;

struct Table {
    void* ptr[kTable];
    int64_t numel[kTable];
    uint32_t first[kTable + 1];  // chunks in front of each tensor
    uint8_t dtype[kTable];
    int32_t count;
};

struct Chunk {
    void* ptr;
    int32_t n;
    int32_t dtype;
};

// chunk c, of tensor `at` or one behind it; `at` follows
template <int CHUNK>
__device__ __forceinline__ Chunk find_chunk(const Table& t, uint32_t c, int& at) {
    if (t.first[at + 1] <= c) {
        int low = at + 1, high = t.count - 1;
        while (low < high) {
            const int mid = (low + high + 1) / 2;
            if (t.first[mid] <= c) low = mid;
            else high = mid - 1;
        }
        at = low;
    }
    const int64_t begin = (int64_t)(c - t.first[at]) * CHUNK, rest = t.numel[at] - begin;
    const int dtype = t.dtype[at];
    Chunk out;
    out.ptr = (char*)t.ptr[at] + begin * (dtype == FMA_F32 ? 4 : 2);
    out.n = (int32_t)(rest < CHUNK ? rest : CHUNK);
    out.dtype = dtype;
    return out;
}

// elements in front of the first 16-byte boundary
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
    const int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    return head < n ? head : n;
}

// sum of squares, or the largest magnitude's bits (as those of a float: their order is that of the numbers, with NaN on top)
template <bool MAX>
struct Accumulator {
    double sum = 0.0;
    __device__ __forceinline__ void add(float x) { sum = __builtin_fma((double)x, (double)x, sum); }
    __device__ __forceinline__ void join(uint64_t bits) { sum += __builtin_bit_cast(double, bits); }
    __device__ __forceinline__ uint64_t bits() const { return __builtin_bit_cast(uint64_t, sum); }
};
template <>
struct Accumulator<true> {
    uint32_t most = 0;
    __device__ __forceinline__ void add(float x) { most = max(most, __float_as_uint(x) & 0x7fffffffu); }
    __device__ __forceinline__ void join(uint64_t bits) { most = max(most, (uint32_t)bits); }
    __device__ __forceinline__ uint64_t bits() const { return most; }
};

template <bool MAX, int WAVES>
__device__ __forceinline__ void join_workgroup(Accumulator<MAX>& acc) {
    __shared__ uint64_t s_part[WAVES];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) acc.join(__shfl_xor(acc.bits(), d, kWave));
    if ((threadIdx.x & (kWave - 1)) == 0) s_part[threadIdx.x / kWave] = acc.bits();
    __syncthreads();
    acc = Accumulator<MAX>();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) acc.join(s_part[w]);
}

// The elements of a chunk: those in front of the first 16-byte boundary and behind the last one go to `one`, the vectors between them to
// `many`, UNROLL neighbouring groups of 256 vectors at a time, and one by one what is left of them.
template <int UNROLL, typename T, typename ONE, typename MANY>
__device__ __forceinline__ void over_chunk(T* p, int n, ONE one, MANY many) {
    constexpr int V = Vec16<T>::N;
    const int head = head_of(p, n);
    if ((int)threadIdx.x < head) one(p + threadIdx.x);
    p += head;
    n -= head;
    const int nvec = n / V;
    Vec16<T>* const v = (Vec16<T>*)p;
    int i = threadIdx.x;
    for (; i + (UNROLL - 1) * kThreads < nvec; i += UNROLL * kThreads) many(v + i, std::integral_constant<int, UNROLL>());
    for (; i < nvec; i += kThreads) many(v + i, std::integral_constant<int, 1>());
    const int tail = nvec * V + (int)threadIdx.x;
    if (tail < n) one(p + tail);
}

template <bool STREAM, typename V>
__device__ __forceinline__ V load(const V* p) {
    if constexpr (STREAM) return load_streaming16(p);
    else return *p;
}

template <bool STREAM, typename T, bool MAX>
__device__ __forceinline__ void add_chunk(Accumulator<MAX>& acc, T* p, int n) {
    over_chunk<8>(
        p, n, [&](const T* x) { acc.add(Num<T>::up(*x)); },
        [&](const Vec16<T>* v, auto times) {
            constexpr int U = decltype(times)::value;
            Vec16<T> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = load<STREAM>(v + u * kThreads);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; ++e) acc.add(Num<T>::up(x[u].v[e]));
        });
}

// 2.2 GB of bf16: 323 us, 6.9 TB/s; 18.9 MB in 120 tensors: 7.8 us, most of it launch and latency
template <bool MAX, bool STREAM>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const Table t, uint64_t* __restrict__ partial) {
    Accumulator<MAX> acc;
    int at = 0;
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const Chunk k = find_chunk<kNormChunk>(t, c, at);
        if (k.dtype == FMA_F32) add_chunk<STREAM>(acc, (float*)k.ptr, k.n);
        else if (k.dtype == FMA_F16) add_chunk<STREAM>(acc, (f16_t*)k.ptr, k.n);
        else add_chunk<STREAM>(acc, (bf16_t*)k.ptr, k.n);
    }
    join_workgroup<MAX, kWaves>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc.bits();
}

// the partial results in a fixed order; the norm in 64 bits for the scaling that follows, and in 32 for the caller
constexpr int kJoinThreads = 1024;
template <bool MAX>
__global__ __launch_bounds__(kJoinThreads) void grad_norm_join_kernel(const uint64_t* __restrict__ partial, int64_t count,
                                                                      double* __restrict__ norm64, float* __restrict__ norm) {
    Accumulator<MAX> acc;
    for (int64_t i = threadIdx.x; i < count; i += kJoinThreads) acc.join(partial[i]);
    join_workgroup<MAX, kJoinThreads / kWave>(acc);
    if (threadIdx.x == 0) {
        double n;
        if constexpr (MAX) n = (double)__uint_as_float(acc.most);
        else n = sqrt(acc.sum);
        *norm64 = n;
        *norm = (float)n;
    }
}

// What elements are multiplied by: digits * 2^power. The power is 0 unless the factor lies below float32's normal numbers, where it would have
// few bits or be 0 while the products (2^125 times 2^-135) are ordinary numbers: the digits are then in [1/2, 1), and the power, which is
// applied to the product, rounds only what is itself below the normal numbers. (Against a product alone: 723 / 725 us for 2.2 GB of bf16,
// 9.1 / 9.1 for 18.9 MB of fp32.)
struct Factor {
    float digits;
    int power;
    __device__ __forceinline__ explicit Factor(double f) : digits((float)f), power(0) {
        if (fabs(f) < 0x1p-126) digits = (float)frexp(f, &power);
    }
    __device__ __forceinline__ float times(float x) const { return ldexpf(x * digits, power); }
};

template <bool STREAM, typename T>
__device__ __forceinline__ void scale_chunk(T* p, int n, const Factor& factor) {
    over_chunk<4>(
        p, n, [&](T* x) { *x = Num<T>::down(factor.times(Num<T>::up(*x))); },
        [&](Vec16<T>* v, auto times) {
            constexpr int U = decltype(times)::value;
            Vec16<T> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = load<STREAM>(v + u * kThreads);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; ++e) x[u].v[e] = Num<T>::down(factor.times(Num<T>::up(x[u].v[e])));
                if constexpr (STREAM) store_streaming16(v + u * kThreads, x[u]);
                else v[u * kThreads] = x[u];
            }
        });
}

// A factor of one leaves the tensors alone: nothing is read or written then. A NaN goes through. A workgroup per chunk, which ends with it, keeps more
// loads and stores in flight than workgroups that stay: 2.2 GB of bf16 722 us, 6.1 TB/s (a copy of that size: 4.8, an elementwise product in place 5.9);
// 18.9 MB in 120 tensors 12 us.
template <bool STREAM>
__global__ __launch_bounds__(kThreads) void scale_grads_kernel(const Table t, const double* __restrict__ norm64,
                                                               const float* __restrict__ norm, double max_norm) {
    const double ratio = max_norm / ((norm64 ? *norm64 : (double)*norm) + 1e-6);
    if (ratio >= 1.0) return;
    const Factor factor(ratio);
    int at = 0;
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const Chunk k = find_chunk<kScaleChunk>(t, c, at);
        if (k.dtype == FMA_F32) scale_chunk<STREAM>((float*)k.ptr, k.n, factor);
        else if (k.dtype == FMA_F16) scale_chunk<STREAM>((f16_t*)k.ptr, k.n, factor);
        else scale_chunk<STREAM>((bf16_t*)k.ptr, k.n, factor);
    }
}

int64_t most_workgroups() { return (num_compute_units() > 0 ? num_compute_units() : 256) * (int64_t)kNormPerCU; }

bool streams(const int64_t* sizes, const int32_t* dtypes, int64_t count) {
    int64_t bytes = 0;
    for (int64_t i = 0; i < count && bytes <= kStreamBytes; ++i) bytes += sizes[i] * dtype_bytes(dtypes[i]);
    return bytes > kStreamBytes;
}

// Tables of the tensors that have elements, in order, and what `launch` makes of each; stops at the first that fails.
template <typename F>
int for_each_table(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, int chunk, F launch) {
    Table t;
    int64_t i = 0;
    while (i < count) {
        t.count = 0;
        t.first[0] = 0;
        for (; i < count && t.count < kTable; ++i) {
            if (sizes[i] == 0) continue;
            const int64_t chunks = (sizes[i] + chunk - 1) / chunk;  // 2^24 at the most, of all tensors of a table below 2^32
            t.ptr[t.count] = tensors[i];
            t.numel[t.count] = sizes[i];
            t.dtype[t.count] = (uint8_t)dtypes[i];
            t.first[t.count + 1] = t.first[t.count] + (uint32_t)chunks;
            ++t.count;
        }
        if (t.count > 0) {
            const int rc = launch(t);
            if (rc) return rc;
        }
    }
    return FMA_OK;
}

int check_tensors(const char* what, void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count) {
    FMA_REQUIRE(count >= 0 && count <= FMA_MAX_GRAD_TENSORS, FMA_ERR_BAD_SIZE, "%s: bad number of tensors %lld", what, (long long)count);
    if (count == 0) return FMA_OK;
    FMA_REQUIRE(tensors && sizes && dtypes, FMA_ERR_NULL_POINTER, "%s: NULL pointer", what);
    for (int64_t i = 0; i < count; ++i) {
        const int bytes = dtype_bytes(dtypes[i]);
        FMA_REQUIRE(bytes != 0, FMA_ERR_BAD_DTYPE, "%s: unknown dtype code %d of tensor %lld", what, (int)dtypes[i], (long long)i);
        FMA_REQUIRE(sizes[i] >= 0 && sizes[i] <= FMA_MAX_GRAD_ELEMENTS, FMA_ERR_BAD_SIZE, "%s: bad size %lld of tensor %lld", what,
                    (long long)sizes[i], (long long)i);
        FMA_REQUIRE(sizes[i] == 0 || tensors[i], FMA_ERR_NULL_POINTER, "%s: tensor %lld is NULL", what, (long long)i);
        FMA_REQUIRE(((uintptr_t)tensors[i] & (uintptr_t)(bytes - 1)) == 0, FMA_ERR_MISALIGNED,
                    "%s: tensor %lld is not aligned to its elements", what, (long long)i);
    }
    return FMA_OK;
}

// No element may be scaled twice, least of all by two workgroups at once, nor the norm that all of them read.
int check_disjoint(const char* what, void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, const void* norm,
                   size_t norm_bytes) {
    struct Range {
        uintptr_t begin, end;
    };
    Range* const r = (Range*)malloc((size_t)(count > 0 ? count : 1) * sizeof(Range));
    FMA_REQUIRE(r, FMA_ERR_BAD_SIZE, "%s: no host memory for %lld tensors", what, (long long)count);
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i)
        if (sizes[i] > 0) {
            r[n].begin = (uintptr_t)tensors[i];
            r[n++].end = (uintptr_t)tensors[i] + (uintptr_t)sizes[i] * (uintptr_t)dtype_bytes(dtypes[i]);
        }
    const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
    if (!std::is_sorted(r, r + n, before)) std::sort(r, r + n, before);  // (those of a bucket are)
    bool apart = true, outside = true;
    for (int64_t i = 1; i < n; ++i) apart = apart && r[i - 1].end <= r[i].begin;
    const uintptr_t at = (uintptr_t)norm;
    for (int64_t i = 0; i < n; ++i) outside = outside && (r[i].end <= at || at + norm_bytes <= r[i].begin);
    free(r);
    FMA_REQUIRE(apart, FMA_ERR_UNSUPPORTED, "%s: two tensors share memory", what);
    FMA_REQUIRE(outside, FMA_ERR_UNSUPPORTED, "%s: the norm shares memory with a tensor", what);
    return FMA_OK;
}

int launch_norm(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, int infinity, float* norm, double* norm64,
                hipStream_t st) {
    uint64_t* const partial = (uint64_t*)(norm64 + 1);
    const int64_t most = most_workgroups();
    int64_t parts = 0;
    const bool stream = streams(sizes, dtypes, count);
    int rc = for_each_table(tensors, sizes, dtypes, count, kNormChunk, [&](const Table& t) {
        const int64_t chunks = t.first[t.count], grid = chunks < most ? chunks : most;
        const auto kernel = infinity ? (stream ? grad_norm_kernel<true, true> : grad_norm_kernel<true, false>)
                                     : (stream ? grad_norm_kernel<false, true> : grad_norm_kernel<false, false>);
        hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(kThreads), 0, st, t, partial + parts);
        parts += grid;
        return launch_status("grad_norm");
    });
    if (rc) return rc;
    if (infinity) hipLaunchKernelGGL(grad_norm_join_kernel<true>, dim3(1), dim3(kJoinThreads), 0, st, partial, parts, norm64, norm);
    else hipLaunchKernelGGL(grad_norm_join_kernel<false>, dim3(1), dim3(kJoinThreads), 0, st, partial, parts, norm64, norm);
    return launch_status("grad_norm (join)");
}

int launch_scale(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, const double* norm64, const float* norm,
                 double max_norm, hipStream_t st) {
    const auto kernel = streams(sizes, dtypes, count) ? scale_grads_kernel<true> : scale_grads_kernel<false>;
    return for_each_table(tensors, sizes, dtypes, count, kScaleChunk, [&](const Table& t) {
        const int64_t chunks = t.first[t.count], grid = chunks < kMostGrid ? chunks : kMostGrid;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(kThreads), 0, st, t, norm64, norm, max_norm);
        return launch_status("scale_grads");
    });
}

int check_workspace(const char* what, const void* workspace, int64_t bytes, int64_t count) {
    FMA_REQUIRE(workspace, FMA_ERR_NULL_POINTER, "%s: NULL workspace", what);
    const int64_t need = fma_grad_norm_workspace_bytes(count);
    FMA_REQUIRE(bytes >= need, FMA_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes,
                (long long)need);
    FMA_REQUIRE(((uintptr_t)workspace & 7u) == 0, FMA_ERR_MISALIGNED, "%s: workspace must be 8-byte aligned", what);
    return FMA_OK;
}

int check_bound(const char* what, double max_norm) {
    FMA_REQUIRE(max_norm >= 0.0, FMA_ERR_BAD_SIZE, "%s: max_norm must not be negative or NaN", what);
    return FMA_OK;
}

int check_scale(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, const void* norm, size_t norm_bytes,
                double max_norm) {
    int rc = check_tensors("scale_grads", tensors, sizes, dtypes, count);
    if (!rc) rc = check_bound("scale_grads", max_norm);
    if (rc) return rc;
    FMA_REQUIRE(norm, FMA_ERR_NULL_POINTER, "scale_grads: norm is NULL");
    FMA_REQUIRE(((uintptr_t)norm & (norm_bytes - 1)) == 0, FMA_ERR_MISALIGNED, "scale_grads: norm is not aligned to its %d bytes",
                (int)norm_bytes);
    return check_disjoint("scale_grads", tensors, sizes, dtypes, count, norm, norm_bytes);
}

}  // namespace
}  // namespace fmahip

extern "C" {

int64_t fma_grad_norm_workspace_bytes(int64_t count) {
    if (count < 0 || count > FMA_MAX_GRAD_TENSORS) return 0;
    // the norm in 64 bits, and a partial result per workgroup of every launch
    return 8 + 8 * fmahip::most_workgroups() * ((count + fmahip::kTable - 1) / fmahip::kTable);
}

int fma_grad_norm(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, int infinity, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace fmahip;
    int rc = check_tensors("grad_norm", tensors, sizes, dtypes, count);
    if (rc) return rc;
    FMA_REQUIRE(norm, FMA_ERR_NULL_POINTER, "grad_norm: norm is NULL");
    rc = check_workspace("grad_norm", workspace, workspace_bytes, count);
    if (rc) return rc;
    return launch_norm(tensors, sizes, dtypes, count, infinity, norm, (double*)workspace, (hipStream_t)stream);
}

int fma_scale_grads(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, const float* norm, double max_norm,
                    void* stream) {
    using namespace fmahip;
    const int rc = check_scale(tensors, sizes, dtypes, count, norm, sizeof(*norm), max_norm);
    return rc ? rc : launch_scale(tensors, sizes, dtypes, count, nullptr, norm, max_norm, (hipStream_t)stream);
}

int fma_scale_grads_norm64(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, const double* norm,
                           double max_norm, void* stream) {
    using namespace fmahip;
    const int rc = check_scale(tensors, sizes, dtypes, count, norm, sizeof(*norm), max_norm);
    return rc ? rc : launch_scale(tensors, sizes, dtypes, count, norm, nullptr, max_norm, (hipStream_t)stream);
}

int fma_clip_grad_norm(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t count, int infinity, double max_norm,
                       float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace fmahip;
    int rc = check_tensors("clip_grad_norm", tensors, sizes, dtypes, count);
    if (!rc) rc = check_bound("clip_grad_norm", max_norm);
    if (rc) return rc;
    FMA_REQUIRE(norm, FMA_ERR_NULL_POINTER, "clip_grad_norm: norm is NULL");
    rc = check_disjoint("clip_grad_norm", tensors, sizes, dtypes, count, norm, sizeof(*norm));
    if (rc) return rc;
    rc = check_workspace("clip_grad_norm", workspace, workspace_bytes, count);
    if (!rc) rc = launch_norm(tensors, sizes, dtypes, count, infinity, norm, (double*)workspace, (hipStream_t)stream);
    if (!rc) rc = launch_scale(tensors, sizes, dtypes, count, (const double*)workspace, nullptr, max_norm, (hipStream_t)stream);
    return rc;
}

}  // extern "C"
