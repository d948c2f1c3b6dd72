"""`fused_sandwich_rmsnorm`: what a transformer block with a norm on either side does at its end, in one pass over the rows:

    stream = residual + multiplier * gate * rms_norm(x) * post_weight
    output = rms_norm(stream) * weight                                    the next block's input

The reference has no counterpart; its fused_residual_add_rmsnorm (fma/ops/fused_residual_add_rmsnorm/__init__.py) is the block's end without
the norm behind it."""

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ...kernel_backend import KernelBackend, is_hip_kernel_backend
from .cuda_implementation import fused_sandwich_rmsnorm_backward_cuda, fused_sandwich_rmsnorm_forward_cuda

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def gate_rows(gate: torch.Tensor, x: torch.Tensor) -> int:
    """How many rows the gate has; each serves the same number of neighbouring rows of x. Raises AssertionError for any other gate."""
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    fits = gate.dim() <= x.dim() and shape[-1] in (1, x.size(-1))
    # from the left: dimensions of x, then ones
    rows, shared = 1, False
    for n, m in zip(shape[:-1], x.shape[:-1]) if fits else ():
        fits = fits and n in (1, m) and not (shared and n > 1)
        shared = shared or n != m
        rows *= n
    assert fits, (
        f"a gate of shape {tuple(gate.shape)} does not fit x of shape {tuple(x.shape)}: its leading dimensions should be those of x up to some "
        "point and 1 from there on, its last one 1 or that of x"
    )
    return rows


def _forward(x, residual, post_weight, weight, gate, rows_of_gate, eps, multiplier, keep):
    """the outputs, and what a backward pass needs of the inputs if one follows (keep)"""
    x, residual, post_weight, weight, gate = [t if t is None else t.contiguous() for t in (x, residual, post_weight, weight, gate)]
    output, stream = torch.empty_like(x), torch.empty_like(x)
    # 1 / rms of every row of x and of the stream
    stats = torch.empty(2, x.numel() // x.size(-1), dtype=torch.float32, device=x.device) if keep else None
    fused_sandwich_rmsnorm_forward_cuda(x, residual, post_weight, weight, gate, output, stream, stats, rows_of_gate, eps, multiplier)
    return (output, stream), (x, residual, post_weight, weight, gate, stats) if keep else None


class _FusedSandwichRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, post_weight, weight, gate, rows_of_gate, eps, multiplier, grad_enabled):
        keep = grad_enabled and any(ctx.needs_input_grad)
        outputs, kept = _forward(x, residual, post_weight, weight, gate, rows_of_gate, eps, multiplier, keep)
        if keep:
            ctx.save_for_backward(*kept)
            ctx.rows_of_gate, ctx.multiplier = rows_of_gate, multiplier
        ctx.set_materialize_grads(False)
        return outputs

    @staticmethod
    @once_differentiable
    def backward(ctx, output_grad, stream_grad):
        if output_grad is None and stream_grad is None:
            return (None,) * 9
        x, residual, post_weight, weight, gate, stats = ctx.saved_tensors
        output_grad, stream_grad = [t if t is None else t.contiguous() for t in (output_grad, stream_grad)]
        x_grad, residual_grad = torch.empty_like(x), torch.empty_like(x)
        rows = x.numel()
        # (without rows the sums over them are zero)
        new = torch.empty_like if rows else torch.zeros_like
        post_weight_grad, weight_grad, gate_grad = [new(t) if n else None for t, n in zip((post_weight, weight, gate), ctx.needs_input_grad[2:5])]
        if rows:
            fused_sandwich_rmsnorm_backward_cuda(
                x, residual, post_weight, weight, gate, output_grad, stream_grad, stats, x_grad, residual_grad, post_weight_grad, weight_grad,
                gate_grad, ctx.rows_of_gate, ctx.multiplier,
            )  # fmt: skip
        return x_grad, residual_grad, post_weight_grad, weight_grad, gate_grad, None, None, None, None


def fused_sandwich_rmsnorm(
    x: torch.Tensor,
    residual: torch.Tensor,
    post_weight: torch.Tensor | None,
    weight: torch.Tensor | None,
    eps: float | None,
    gate: torch.Tensor | None = None,
    multiplier: float | None = None,
    kernel_backend: KernelBackend = KernelBackend.triton,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Returns (the next block's normalised input, the updated residual stream), both shaped and typed like x.

    x: the block's output; residual: the stream of the same shape; float32, float16 or bfloat16, rows along the last dimension, at most 65536
    long. post_weight, weight: 1-D scales of the norm behind the block and of the one before the next, or None. eps: added to both mean
    squares; None takes the dtype's machine epsilon. gate: multiplies the normed output; of x's dtype and, from the left, of x's dimensions up
    to some point and 1 from there on, the last one 1 or x's (dimensions of 1 may be left out in front): a scale per element (x's shape), per
    channel ([H]), per token ([.., 1]), per sequence and channel ([batch, 1, H]), or a single number. multiplier: the residual scale; None means 1.
    Arithmetic is in float32 with one rounding per output; the second norm is taken of the unrounded stream, in the backward pass too (once; no
    second derivatives), which keeps x, residual, gate, the scales and two numbers per row. kernel_backend: `triton` (the default) and `cuda` both run the HIP
    kernels; anything else raises ValueError.
    """
    if not is_hip_kernel_backend(kernel_backend):
        raise ValueError(f"unexpected kernel_backend ({kernel_backend})")
    assert x.dtype in _FLOATS, f"fused_sandwich_rmsnorm takes float32, float16 and bfloat16, not {x.dtype}"
    assert x.dim() >= 1 and x.size(-1) > 0, "x should have rows of one element at least"
    rows = 0
    if gate is not None:
        assert gate.dtype == x.dtype, "gate should have x's dtype"
        rows = gate_rows(gate, x)
    # (the operator looks at the other tensors)
    eps = torch.finfo(x.dtype).eps if eps is None else float(eps)
    arguments = x, residual, post_weight, weight, gate, rows, eps, 1.0 if multiplier is None else float(multiplier)
    grad_enabled = torch.is_grad_enabled()
    if not grad_enabled and forward_ad._current_level < 0 and not torch._C._are_functorch_transforms_active():
        return _forward(*arguments, False)[0]  # (an autograd node that nothing asks for is 4 us)
    return _FusedSandwichRMSNorm.apply(*arguments, grad_enabled)
