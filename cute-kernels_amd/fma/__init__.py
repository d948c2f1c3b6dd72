"""MI355X-native implementation of the MoE-layer hot path of cute-kernels (`fma`): same public names and call
signatures for the ops and the module on that path, computed by hand-written HIP kernels (gfx950) behind a C ABI."""

from .kernel_backend import KernelBackend
from .math import ceil_divide, divide_if_divisible
from .modules import MoE, quantize_expert_weights, swiglu_experts_fp8
from .ops import (
    Fp8Blocks,
    clip_grad_norm_,
    clip_grads_with_norm_,
    continuous_count,
    dequantize_fp8,
    fused_residual_add_rmsnorm,
    fused_sandwich_rmsnorm,
    get_total_norm,
    grouped_gemm,
    grouped_gemm_fp8,
    grouped_linear_fp8,
    quantize_fp8,
    router_loss,
    swiglu,
    swiglu_packed,
    swiglu_packed_fp8,
)
from .utils import ensure_contiguous, set_seed
