"""The expert path of a SwiGLU layer with its products in 8 bits (fma_swiglu_experts_fp8 and its backward, one call per direction)."""

import torch
from torch.autograd import forward_ad

from ... import _lib
from ..._ops import hip_op
from ...ops.fp8 import BLOCK_SIZE, Fp8Blocks, quantize_fp8
from ...ops.fp8.cuda_implementation import is_scales_dtype, operator_scales, quantize_fp8_cuda
from ...utils import ensure_contiguous


def _check_operands(x, router_weights, selected_experts, weight1, weight1_scales, weight2, weight2_scales):
    """(T, k, E, H, I); weight1 [E, 2, I, H], weight2 [E, H, I]"""
    T, H = x.shape
    E, two, I, _ = weight1.shape
    k = selected_experts.size(1)
    assert two == 2 and weight1.shape == (E, 2, I, H) and weight2.shape == (E, H, I)
    assert selected_experts.shape == router_weights.shape == (T, k) and selected_experts.dtype in (torch.int32, torch.int64)
    assert x.dtype == router_weights.dtype and x.dtype in (torch.float16, torch.bfloat16)
    for values, scales in ((weight1, weight1_scales), (weight2, weight2_scales)):
        assert values.dtype == torch.float8_e4m3fn and is_scales_dtype(scales.dtype)
        N, K = values.shape[-2:]
        assert scales.shape == (*values.shape[:-2], -(-N // 128), 4 * -(-K // 512))
    for t in (x, router_weights, selected_experts, weight1, weight1_scales, weight2, weight2_scales):
        assert t.is_contiguous() and t.device == x.device
    return T, k, E, H, I


@hip_op("swiglu_experts_fp8_cuda", mutates_args={"output", "buffer"})
def swiglu_experts_fp8_cuda(
    x: torch.Tensor, router_weights: torch.Tensor, selected_experts: torch.Tensor, weight1: torch.Tensor, weight1_scales: torch.Tensor,
    weight2: torch.Tensor, weight2_scales: torch.Tensor, output: torch.Tensor, buffer: torch.Tensor | None,
) -> None:  # fmt: skip
    """buffer: what a backward pass reads (buffer_bytes); without it the call owns that memory too"""
    _lib.require_gpu(x, router_weights, selected_experts, weight1, weight1_scales, weight2, weight2_scales, output, buffer)
    T, k, E, H, I = _check_operands(x, router_weights, selected_experts, weight1, weight1_scales, weight2, weight2_scales)
    assert output.shape == (T, H) and output.dtype == x.dtype and output.is_contiguous()
    lib = _lib.load()
    keep = buffer is not None
    with _lib.on_device(x.device):
        if not keep:
            buffer = x.new_empty(lib.fma_swiglu_experts_fp8_buffer_bytes(T, k, E, H, I, 0), dtype=torch.uint8)
        workspace = x.new_empty(lib.fma_swiglu_experts_fp8_workspace_bytes(T, k, E), dtype=torch.uint8)
        rc = lib.fma_swiglu_experts_fp8(
            x.data_ptr(), router_weights.data_ptr(), selected_experts.data_ptr(), selected_experts.element_size(), weight1.data_ptr(),
            weight1_scales.data_ptr(), weight2.data_ptr(), weight2_scales.data_ptr(), output.data_ptr(), T, k, E, H, I, int(keep),
            buffer.data_ptr(), buffer.numel(), workspace.data_ptr(), workspace.numel(), _lib.dtype_code(x.dtype),
            _lib.current_stream(x.device),
        )  # fmt: skip
    _lib.check(rc, "swiglu_experts_fp8_cuda")


@hip_op("swiglu_experts_fp8_backward_cuda", mutates_args={"x_grad", "router_weights_grad", "weight1_grad", "weight2_grad"})
def swiglu_experts_fp8_backward_cuda(
    output_grad: torch.Tensor, router_weights: torch.Tensor, selected_experts: torch.Tensor, weight1_t: torch.Tensor,
    weight1_t_scales: torch.Tensor, weight2_t: torch.Tensor, weight2_t_scales: torch.Tensor, buffer: torch.Tensor,
    x_grad: torch.Tensor | None, router_weights_grad: torch.Tensor | None, weight1_grad: torch.Tensor | None,
    weight2_grad: torch.Tensor | None,
) -> None:  # fmt: skip
    """weight1_t [E, 2, H, I], weight2_t [E, I, H]: the transposed copies"""
    grads = (x_grad, router_weights_grad, weight1_grad, weight2_grad)
    _lib.require_gpu(output_grad, router_weights, selected_experts, weight1_t, weight1_t_scales, weight2_t, weight2_t_scales, buffer, *grads)
    T, H = output_grad.shape
    E, I, _ = weight2_t.shape
    k = selected_experts.size(1)
    assert weight1_t.shape == (E, 2, H, I) and weight2_t.shape == (E, I, H)
    assert selected_experts.shape == router_weights.shape == (T, k) and output_grad.dtype == router_weights.dtype
    for t in (output_grad, router_weights, selected_experts, weight1_t, weight1_t_scales, weight2_t, weight2_t_scales, buffer):
        assert t.is_contiguous() and t.device == output_grad.device
    for t, shape in zip(grads, ((T, H), (T, k), (E, 2 * I, H), (E, H, I))):
        assert t is None or (t.shape == shape and t.dtype == output_grad.dtype and t.is_contiguous())
    lib = _lib.load()
    with _lib.on_device(output_grad.device):
        workspace = output_grad.new_empty(lib.fma_swiglu_experts_fp8_bwd_workspace_bytes(T, k, H, I), dtype=torch.uint8)
        rc = lib.fma_swiglu_experts_fp8_bwd(
            output_grad.data_ptr(), router_weights.data_ptr(), selected_experts.data_ptr(), selected_experts.element_size(),
            weight1_t.data_ptr(), weight1_t_scales.data_ptr(), weight2_t.data_ptr(), weight2_t_scales.data_ptr(), buffer.data_ptr(),
            buffer.numel(), *[_lib.ptr(t) for t in grads], T, k, E, H, I, workspace.data_ptr(), workspace.numel(),
            _lib.dtype_code(output_grad.dtype), _lib.current_stream(output_grad.device),
        )  # fmt: skip
    _lib.check(rc, "swiglu_experts_fp8_backward_cuda")


def buffer_bytes(T: int, k: int, E: int, H: int, I: int) -> int:
    """fma_swiglu_experts_fp8_buffer_bytes with keep, where a traced layer can compute it: tokens, activation and pre-activation in 8 bits
    with their scales, the experts' output, sizes and offsets of the experts, the routing order and its inverse"""
    R, scales_H, scales_I = T * k, 4 * -(-H // 512), 4 * -(-I // 512)
    pieces = (T * H, T * scales_H, R * I, R * scales_I, 2 * R * H, 4 * E, 4 * E, 4 * R, 4 * R, 2 * R * I, 2 * R * scales_I)
    return sum(-(-n // 256) * 256 for n in pieces)


def quantize_expert_weights(
    weight1: torch.Tensor, weight2: torch.Tensor, transposed: bool = False
) -> tuple[Fp8Blocks, Fp8Blocks] | tuple[tuple[Fp8Blocks, Fp8Blocks], tuple[Fp8Blocks, Fp8Blocks]]:
    """The projections of a SwiGLU layer's experts in 128 x 128 blocks: weight1 [E, 2 I, H] as [E, 2, I, H] (the up and the gate projection
    are matrices of their own) and weight2 [E, H, I]. transposed: each with its transposed copy."""
    E, two_I, H = weight1.shape
    return (
        quantize_fp8(weight1.reshape(E, 2, two_I // 2, H), BLOCK_SIZE, transposed),
        quantize_fp8(weight2, BLOCK_SIZE, transposed),
    )


def requantize_expert_weights(weight1: torch.Tensor, weight2: torch.Tensor, blocks1: Fp8Blocks, blocks2: Fp8Blocks) -> None:
    """quantize_expert_weights into the blocks that it has given for weights of the same shapes"""
    for weight, blocks in ((weight1, blocks1), (weight2, blocks2)):
        quantize_fp8_cuda(weight.detach().contiguous().view(blocks.values.shape), *blocks, None, None, BLOCK_SIZE)


class _SwigluExpertsFp8(torch.autograd.Function):
    @staticmethod
    @ensure_contiguous
    def forward(
        ctx, x: torch.Tensor, router_weights: torch.Tensor, selected_experts: torch.Tensor, weight1: torch.Tensor, weight2: torch.Tensor,
        grad_enabled: bool,
    ) -> torch.Tensor:  # fmt: skip
        T, H = x.shape
        E, two_I, _ = weight1.shape
        needs = [grad_enabled and n for n in ctx.needs_input_grad]
        keeps = any(needs)
        ctx.weight_shapes = weight1.shape, weight2.shape
        if not keeps:
            c_fc, c_proj = quantize_expert_weights(weight1, weight2)
        else:
            (c_fc, c_fc_t), (c_proj, c_proj_t) = quantize_expert_weights(weight1, weight2, transposed=True)
        output = torch.empty_like(x)
        buffer = None
        if keeps:
            buffer = x.new_empty(buffer_bytes(T, selected_experts.size(1), E, H, two_I // 2), dtype=torch.uint8)
        if T:
            operands = c_fc[0], operator_scales(c_fc[1]), c_proj[0], operator_scales(c_proj[1])
            swiglu_experts_fp8_cuda(x, router_weights, selected_experts, *operands, output, buffer)
        if keeps:
            operands = c_fc_t[0], operator_scales(c_fc_t[1]), c_proj_t[0], operator_scales(c_proj_t[1])
            ctx.save_for_backward(router_weights, selected_experts, *operands, buffer)
        return output

    @staticmethod
    @ensure_contiguous
    def backward(ctx, output_grad: torch.Tensor) -> tuple[torch.Tensor | None, ...]:
        router_weights, selected_experts, *weights, buffer = ctx.saved_tensors
        needs_x, needs_gates, _, needs_weight1, needs_weight2, _ = ctx.needs_input_grad
        make = output_grad.new_empty if output_grad.size(0) else output_grad.new_zeros
        x_grad = torch.empty_like(output_grad) if needs_x else None
        gates_grad = torch.empty_like(router_weights) if needs_gates else None
        weight1_grad = make(ctx.weight_shapes[0]) if needs_weight1 else None
        weight2_grad = make(ctx.weight_shapes[1]) if needs_weight2 else None
        if output_grad.size(0):
            swiglu_experts_fp8_backward_cuda(
                output_grad, router_weights, selected_experts, *weights, buffer, x_grad, gates_grad, weight1_grad, weight2_grad
            )
        return x_grad, gates_grad, None, weight1_grad, weight2_grad, None


def swiglu_experts_fp8(
    x: torch.Tensor,
    router_weights: torch.Tensor,
    selected_experts: torch.Tensor,
    c_fc: torch.Tensor | Fp8Blocks,
    c_proj: torch.Tensor | Fp8Blocks,
) -> torch.Tensor:
    """The experts of a SwiGLU layer with their products in 8 bits: for every token the sum, weighted with router_weights [T, k], of
    swiglu(x W1_e^T) W2_e^T over its selected_experts [T, k] (int32 or int64; an id that names no expert contributes nothing).

    x [T, H] and router_weights: float16 or bfloat16. c_fc [E, 2 I, H] ("up" rows, then "gate" rows) and c_proj [E, H, I]: either 16-bit
    tensors of x's dtype, quantised in the call, with gradients for all four; or, for serving, what quantize_expert_weights has made of
    them, without gradients (a call that would need one is refused). x, the pre-activation and the activation are quantised in blocks of 128
    along their rows, and a training step keeps them in that form. H and I must be multiples of 16.

    Activations past float16's range are held as they are, in the gradients too; tokens and pre-activations of 248 * 2^120 and more, 2^128 in
    8 bits, may count as infinite. Sums that are rounded to 8 bits again are exact to fp32 in a training step's forward pass and for a few tokens, and cut
    at 2^-13 of the largest of eight products otherwise: results of the three differ by up to 0.003 of their norm."""
    assert x.dim() == 2 and selected_experts.dim() == 2, "x should be [T, H], selected_experts [T, k]"
    assert router_weights.shape == selected_experts.shape and selected_experts.size(0) == x.size(0), "one weight per choice of a token"
    assert x.dtype in (torch.float16, torch.bfloat16) and router_weights.dtype == x.dtype, "tokens and weights in float16 or bfloat16"
    assert selected_experts.dtype in (torch.int32, torch.int64), "selected_experts should be int32 or int64"
    assert selected_experts.size(1) > 0, "every token should have a choice"
    prepared = isinstance(c_fc, tuple)
    assert prepared == isinstance(c_proj, tuple), "both projections in 8 bits, or neither"
    H = x.size(1)
    if prepared:
        assert c_fc[0].dim() == 4 and c_fc[0].size(1) == 2 and c_proj[0].dim() == 3, "c_fc should be [E, 2, I, H], c_proj [E, H, I]"
        E, _, I, _ = c_fc[0].shape
        assert c_fc[0].shape == (E, 2, I, H) and c_proj[0].shape == (E, H, I), "sizes of tokens and projections should agree"
    else:
        assert c_fc.dim() == 3 and c_proj.dim() == 3 and c_fc.size(1) % 2 == 0, "c_fc should be [E, 2 I, H], c_proj [E, H, I]"
        E, I = c_fc.size(0), c_fc.size(1) // 2
        assert c_fc.shape == (E, 2 * I, H) and c_proj.shape == (E, H, I), "sizes of tokens and projections should agree"
        assert c_fc.dtype == c_proj.dtype == x.dtype, "projections in 16 bits should have the tokens' dtype"
    assert E > 0, "there should be an expert"
    assert H > 0 and I > 0 and H % 16 == 0 and I % 16 == 0, "hidden and intermediate size should be multiples of 16"
    if not prepared:
        return _SwigluExpertsFp8.apply(x, router_weights, selected_experts, c_fc, c_proj, torch.is_grad_enabled())
    tangents = forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, router_weights))
    if tangents or (torch.is_grad_enabled() and (x.requires_grad or router_weights.requires_grad)):
        raise RuntimeError("swiglu_experts_fp8 has no gradients through projections that are in 8 bits already: pass the 16-bit tensors")
    with torch.no_grad():
        x, router_weights, selected_experts = x.contiguous(), router_weights.contiguous(), selected_experts.contiguous()
        output = torch.empty_like(x)
        if x.size(0):
            c_fc, c_fc_scales, c_proj, c_proj_scales = (t.contiguous() for t in (*c_fc, *c_proj))
            operands = c_fc, operator_scales(c_fc_scales), c_proj, operator_scales(c_proj_scales)
            swiglu_experts_fp8_cuda(x, router_weights, selected_experts, *operands, output, None)
        return output
