// Products of 8-bit weights with a few rows per group (a decode step), for the sources that launch them (fp8_thin.hip has the kernels).
#pragma once

#include "fp8_parts.h"

namespace fmahip {
namespace fp8 {

constexpr int64_t kMaxThinSlots = 1024;  // (token, choice) slots that a workgroup looks through for the rows of its expert

// Whether a product of R rows [R, K] in E groups runs on the kernel for few rows (measured in fp8_thin.hip), and both products of a layer's
// experts do
bool is_thin_product(int64_t E, int64_t R, int64_t N, int64_t K);
bool are_thin_experts(int64_t E, int64_t R, int64_t H, int64_t I);

// D_e = A_e B_e^T as fma_grouped_gemm_fp8, all arguments checked
int launch_thin_product(const void* A, const void* A_s, const void* B, const void* B_s, void* D, const uint32_t* sizes, int64_t E, int64_t R,
                        int64_t N, int64_t K, int dtype, hipStream_t st);

// act[slot] = swiglu(q(x[slot / top_k]) W1_e^T) in fp32 [R, I], e the expert of the slot; W1 [E, 2, I, H]; then o[slot] = q(act[slot]) W2_e^T in fp32
// [R, H]. Slots whose id names no expert are left as they are. R <= kMaxThinSlots.
int launch_thin_experts(const void* x, const void* ids, int id_bytes, const void* W1, const void* W1_s, const void* W2, const void* W2_s, float* act,
                        float* o, int64_t T, int64_t top_k, int64_t E, int64_t H, int64_t I, int dtype, hipStream_t st);

}  // namespace fp8
}  // namespace fmahip
