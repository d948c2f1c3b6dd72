// The grouped product of 8-bit operands, for the sources that launch it (fp8_gemm.hip has the kernels).
#pragma once

#include "fp8_gemm.h"

namespace fmahip {
namespace fp8 {

// Rows per group from device memory (args.sizes), R rows at most. The caller has checked pointers and sizes.
int launch_gemm(const char* who, int epilogue, const GemmArgs& args, hipStream_t st);

// limits of a product: the lane offsets into a tile's rows and the tile count stay below 2^31
int check_gemm(const char* who, int64_t E, int64_t R, int64_t N, int64_t K, int64_t segs);

}  // namespace fp8
}  // namespace fmahip
