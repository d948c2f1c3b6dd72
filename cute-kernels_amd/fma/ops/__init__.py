from .continuous_count import continuous_count
from .fp8 import Fp8Blocks, dequantize_fp8, grouped_gemm_fp8, grouped_linear_fp8, quantize_fp8
from .fused_residual_add_rmsnorm import fused_residual_add_rmsnorm
from .grouped_gemm import grouped_gemm
from .swiglu import swiglu, swiglu_packed, swiglu_packed_fp8
