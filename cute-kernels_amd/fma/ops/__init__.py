from .clip_grad_norm import clip_grad_norm_, clip_grads_with_norm_, get_total_norm
from .continuous_count import continuous_count
from .fp8 import Fp8Blocks, dequantize_fp8, grouped_gemm_fp8, grouped_linear_fp8, quantize_fp8
from .fused_residual_add_rmsnorm import fused_residual_add_rmsnorm
from .fused_sandwich_rmsnorm import fused_sandwich_rmsnorm
from .grouped_gemm import grouped_gemm
from .router_loss import router_loss
from .swiglu import swiglu, swiglu_packed, swiglu_packed_fp8
