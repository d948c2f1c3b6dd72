// Launches of the grouped product of 8-bit operands (fp8_gemm.h) and its C entry point.
#include "fp8_gemm_launch.h"
#include "fp8_thin.h"

namespace fmahip {
namespace gemm {
// grouped_gemm_ragged.hip
int weight_gradient(const void* dy, const void* x, void* dW, const uint32_t* sizes, int64_t rows, int64_t E, int64_t M, int64_t N, int dtype,
                    hipStream_t st);
}  // namespace gemm

namespace fp8 {

int check_gemm(const char* who, int64_t E, int64_t R, int64_t N, int64_t K, int64_t segs) {
    FMA_REQUIRE(E >= 0 && R >= 0 && N >= 0 && K >= 1, FMA_ERR_BAD_SIZE, "%s: bad size E=%lld R=%lld N=%lld K=%lld", who, (long long)E,
                (long long)R, (long long)N, (long long)K);
    FMA_REQUIRE(E <= FMA_MAX_GROUPS, FMA_ERR_TOO_MANY_EXPERTS, "%s: E=%lld, at most %d groups", who, (long long)E, FMA_MAX_GROUPS);
    FMA_REQUIRE(K % 16 == 0, FMA_ERR_BAD_SIZE, "%s: rows of whole 16-byte pieces: K=%lld is no multiple of 16", who, (long long)K);
    FMA_REQUIRE(K < (1 << 21) && N < (1 << 21) && R < (1ll << 31), FMA_ERR_TOO_MANY_ELEMENTS, "%s: K < 2^21, N < 2^21, R < 2^31", who);
    const int64_t row_tiles = R / kTileM + E + 1, col_tiles = (N + kTileN / 2 - 1) / (kTileN / 2);
    FMA_REQUIRE(row_tiles * col_tiles < (1ll << 30), FMA_ERR_TOO_MANY_ELEMENTS, "%s: more than 2^30 tiles", who);
    FMA_REQUIRE(segs * N * K < (1ll << 32), FMA_ERR_TOO_MANY_ELEMENTS, "%s: a group's matrix has 2^32 bytes or more", who);
    return FMA_OK;
}

int launch_gemm(const char* who, int epilogue, const GemmArgs& args, hipStream_t st) {
    const bool glu = epilogue == EPI_GLU || epilogue == EPI_GLU_KEEP;
    const int64_t cols = glu ? kTileN / 2 : kTileN;
    // the host does not know the sizes: as many workgroups as the rows could make tiles, or one per compute unit
    const int64_t tiles = ((int64_t)args.R / kTileM + (args.E < args.R ? args.E : args.R)) * ((args.N + cols - 1) / cols);
    const int64_t cus = num_compute_units() > 0 ? num_compute_units() : 256;
    const dim3 grid((uint32_t)(tiles < cus ? tiles : cus)), block(kGemmThreads);
    const bool tall = args.E <= kTallGroups;
    auto run = [&](auto low, auto high) {
        if (tall) hipLaunchKernelGGL(high, grid, block, 0, st, args);
        else hipLaunchKernelGGL(low, grid, block, 0, st, args);
    };
#define FMA_FP8_RUN(EPI) run(fp8_gemm_kernel<EPI, false>, fp8_gemm_kernel<EPI, true>)
    switch (epilogue) {
        case EPI_BF16: FMA_FP8_RUN(EPI_BF16); break;
        case EPI_F16: FMA_FP8_RUN(EPI_F16); break;
        case EPI_F32: FMA_FP8_RUN(EPI_F32); break;
        case EPI_GLU: FMA_FP8_RUN(EPI_GLU); break;
        case EPI_GLU_KEEP: FMA_FP8_RUN(EPI_GLU_KEEP); break;
        case EPI_GLU_BWD_BF16: FMA_FP8_RUN(EPI_GLU_BWD_BF16); break;
        default: FMA_FP8_RUN(EPI_GLU_BWD_F16); break;
    }
#undef FMA_FP8_RUN
    return launch_status(who);
}

}  // namespace fp8
}  // namespace fmahip

extern "C" {

int fma_grouped_gemm_fp8(const void* A, const void* A_scales, const void* B, const void* B_scales, void* D, const uint32_t* M_arr, int64_t E,
                         int64_t R, int64_t N, int64_t K, int dtype, void* stream) {
    using namespace fmahip;
    using namespace fmahip::fp8;
    FMA_REQUIRE(dtype_bytes(dtype) != 0, FMA_ERR_BAD_DTYPE, "grouped_gemm_fp8: dtype code %d", dtype);
    if (const int rc = check_gemm("grouped_gemm_fp8", E, R, N, K, 1)) return rc;
    FMA_REQUIRE(M_arr || E <= 1, FMA_ERR_NULL_POINTER, "grouped_gemm_fp8: M_arr is NULL, and there are %lld groups", (long long)E);
    if (E == 0 || R == 0 || N == 0) return FMA_OK;
    FMA_REQUIRE(A && A_scales && B && B_scales && D, FMA_ERR_NULL_POINTER, "grouped_gemm_fp8: an operand is NULL");
    FMA_REQUIRE(aligned16(A) && aligned16(B) && aligned16(D), FMA_ERR_MISALIGNED, "grouped_gemm_fp8: A, B and D must be aligned to 16 bytes");
    FMA_REQUIRE(((reinterpret_cast<uintptr_t>(A_scales) | reinterpret_cast<uintptr_t>(B_scales)) & 3u) == 0, FMA_ERR_MISALIGNED,
                "grouped_gemm_fp8: scales must be aligned to 4 bytes");
    if (is_thin_product(E, R, N, K)) return launch_thin_product(A, A_scales, B, B_scales, D, M_arr, E, R, N, K, dtype, (hipStream_t)stream);
    GemmArgs a = {};
    a.A = (const uint8_t*)A;
    a.A_s = (const uint8_t*)A_scales;
    a.B = (const uint8_t*)B;
    a.B_s = (const uint8_t*)B_scales;
    a.sizes = M_arr;
    a.E = (uint32_t)E;
    a.R = (uint32_t)R;
    a.N = (uint32_t)N;
    a.K = (uint32_t)K;
    a.segs = 1;
    a.a_pitch = (uint32_t)K;
    a.as_pitch = a.bs_pitch = (uint32_t)scale_pitch(K);
    a.b_group = (uint64_t)N * K;
    a.bs_group = (uint64_t)((N + kBlock - 1) / kBlock) * a.bs_pitch;
    a.D = D;
    return launch_gemm("grouped_gemm_fp8", dtype == FMA_F32 ? EPI_F32 : (dtype == FMA_F16 ? EPI_F16 : EPI_BF16), a, (hipStream_t)stream);
}

// ---- the product of 16-bit tensors, quantised on the way, and its gradients ----

int fma_grouped_linear_fp8(const void* x, const void* W, void* x_values, void* x_scales, void* W_values, void* W_scales, void* Wt_values,
                           void* Wt_scales, void* y, const uint32_t* M_arr, int64_t E, int64_t R, int64_t N, int64_t K, int dtype,
                           void* stream) {
    using namespace fmahip;
    FMA_REQUIRE(dtype == FMA_BF16 || dtype == FMA_F16, FMA_ERR_BAD_DTYPE, "grouped_linear_fp8: 16-bit tensors only, got dtype code %d", dtype);
    if (const int rc = fmahip::fp8::check_gemm("grouped_linear_fp8", E, R, N, K, 1)) return rc;
    if (const int rc = fma_quantize_fp8(W, W_values, W_scales, Wt_values, Wt_scales, E, N, K, 128, dtype, stream)) return rc;
    if (const int rc = fma_quantize_fp8(x, x_values, x_scales, nullptr, nullptr, 1, R, K, 1, dtype, stream)) return rc;
    return fma_grouped_gemm_fp8(x_values, x_scales, W_values, W_scales, y, M_arr, E, R, N, K, dtype, stream);
}

int64_t fma_grouped_linear_fp8_bwd_workspace_bytes(int64_t R, int64_t N, int64_t K) {
    if (R < 0 || N < 1 || K < 1) return 0;
    auto whole = [](int64_t n) { return (n + 255) & ~(int64_t)255; };
    return whole(R * N) + whole(R * fmahip::fp8::scale_pitch(N)) + whole(R * K * 2);
}

int fma_grouped_linear_fp8_bwd(const void* dy, const void* x_values, const void* x_scales, const void* Wt_values, const void* Wt_scales,
                               void* dx, void* dW, const uint32_t* M_arr, int64_t E, int64_t R, int64_t N, int64_t K, void* workspace,
                               int64_t workspace_bytes, int dtype, void* stream) {
    using namespace fmahip;
    FMA_REQUIRE(dtype == FMA_BF16 || dtype == FMA_F16, FMA_ERR_BAD_DTYPE, "grouped_linear_fp8_bwd: 16-bit tensors only, got dtype code %d", dtype);
    if (const int rc = fmahip::fp8::check_gemm("grouped_linear_fp8_bwd", E, R, K, N, 1)) return rc;
    if (E == 0 || R == 0 || N == 0) return FMA_OK;
    FMA_REQUIRE(dy && M_arr && workspace && (!dx || (Wt_values && Wt_scales)) && (!dW || (x_values && x_scales)), FMA_ERR_NULL_POINTER,
                "grouped_linear_fp8_bwd: a tensor is NULL");
    FMA_REQUIRE(aligned16(dy) && aligned16(workspace) && aligned16(dx) && aligned16(dW), FMA_ERR_MISALIGNED,
                "grouped_linear_fp8_bwd: tensors must be aligned to 16 bytes");
    const int64_t needed = fma_grouped_linear_fp8_bwd_workspace_bytes(R, N, K);
    FMA_REQUIRE(workspace_bytes >= needed, FMA_ERR_WORKSPACE_TOO_SMALL, "grouped_linear_fp8_bwd: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)needed);
    uint8_t* const dy8 = (uint8_t*)workspace;
    uint8_t* const dy8_s = dy8 + ((R * N + 255) & ~(int64_t)255);
    uint8_t* const x16 = dy8_s + ((R * fmahip::fp8::scale_pitch(N) + 255) & ~(int64_t)255);
    if (dx) {
        if (const int rc = fma_quantize_fp8(dy, dy8, dy8_s, nullptr, nullptr, 1, R, N, 1, dtype, stream)) return rc;
        if (const int rc = fma_grouped_gemm_fp8(dy8, dy8_s, Wt_values, Wt_scales, dx, M_arr, E, R, K, N, dtype, stream)) return rc;
    }
    if (dW) {
        if (const int rc = fma_dequantize_fp8(x_values, x_scales, x16, 1, R, K, 1, dtype, stream)) return rc;
        return gemm::weight_gradient(dy, x16, dW, M_arr, R, E, N, K, dtype, (hipStream_t)stream);
    }
    return FMA_OK;
}

}  // extern "C"
