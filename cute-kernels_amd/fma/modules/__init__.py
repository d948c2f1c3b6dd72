from .moe import MoE
from .moe.fp8_implementation import quantize_expert_weights, swiglu_experts_fp8
