"""`swiglu(gate, up)` and `swiglu_packed(x)`: y = up * gate * sigmoid(gate), with gradients. Public names, keyword
arguments, defaults, the shape / dtype assertions and the ValueError for an unknown backend are those of
fma/ops/swiglu/__init__.py:15-164. A packed input holds [up | gate] along its last dimension (the reference's
`up, gate = x.chunk(2, dim=-1)`, :153). Both forms end in the same two strided HIP kernels (`fma_swiglu_forward`,
`fma_swiglu_backward`): the halves of a packed tensor are passed as views, never copied. `swiglu_packed_fp8(x)` is the
latter with its input kept for the backward pass in 8 bits (`fma_swiglu_fp8_forward`, `fma_swiglu_fp8_backward`)."""

import torch

from ...kernel_backend import KernelBackend, is_hip_kernel_backend
from ...math import ceil_divide, divide_if_divisible
from ...utils import ensure_contiguous
from ..fp8.cuda_implementation import scales_dtype
from .cuda_implementation import swiglu_backward_cuda, swiglu_forward_cuda, swiglu_fp8_backward_cuda, swiglu_fp8_forward_cuda

_BLOCK_SIZE = 1024  # a launch-shape argument of the reference's stubs; the HIP kernels choose their own


def _require_hip(*kernel_backends: KernelBackend) -> None:
    for kernel_backend in kernel_backends:
        if not is_hip_kernel_backend(kernel_backend):
            raise ValueError(f"unexpected kernel_backend ({kernel_backend})")


def _check_packed(x: torch.Tensor) -> None:
    assert x.dim() >= 1 and x.size(-1) > 0 and x.size(-1) % 2 == 0, "the last dimension should be even and not empty"
    assert x.dtype in (torch.float32, torch.float16, torch.bfloat16), f"unsupported dtype {x.dtype}"


def _forward(gate: torch.Tensor, up: torch.Tensor, output: torch.Tensor) -> torch.Tensor:
    swiglu_forward_cuda(gate=gate, up=up, output=output, BLOCK_SIZE=_BLOCK_SIZE)
    return output


def _backward(gate, up, output_grad, gate_grad, up_grad) -> None:
    swiglu_backward_cuda(
        gate=gate, up=up, output_grad=output_grad, gate_grad=gate_grad, up_grad=up_grad, BLOCK_SIZE=_BLOCK_SIZE
    )


class _Swiglu(torch.autograd.Function):
    """Two separate operands of one shape."""

    @staticmethod
    @ensure_contiguous
    def forward(ctx, gate: torch.Tensor, up: torch.Tensor, forward_backend, backward_backend) -> torch.Tensor:
        assert gate.size() == up.size(), "tensors gate and up should have same shape"
        assert gate.type() == up.type(), "tensors gate and up should have same dtype"
        _require_hip(forward_backend, backward_backend)
        ctx.save_for_backward(gate, up)
        return _forward(gate, up, torch.empty_like(gate))

    @staticmethod
    @ensure_contiguous
    def backward(ctx, output_grad: torch.Tensor):
        gate, up = ctx.saved_tensors
        grads = torch.empty_like(gate), torch.empty_like(up)
        _backward(gate, up, output_grad, *grads)
        return (*grads, None, None)


class _SwigluPacked(torch.autograd.Function):
    """One operand whose last dimension is [up | gate]; its gradient is written in the same packing."""

    @staticmethod
    @ensure_contiguous
    def forward(ctx, x: torch.Tensor, forward_backend, backward_backend) -> torch.Tensor:
        _require_hip(forward_backend, backward_backend)
        half = divide_if_divisible(x.size(-1), 2)
        up, gate = x.split(half, dim=-1)
        ctx.save_for_backward(x)
        return _forward(gate, up, x.new_empty(*x.shape[:-1], half))

    @staticmethod
    @ensure_contiguous
    def backward(ctx, output_grad: torch.Tensor):
        (x,) = ctx.saved_tensors
        half = x.size(-1) // 2
        x_grad = torch.empty_like(x)
        up, gate = x.split(half, dim=-1)
        up_grad, gate_grad = x_grad.split(half, dim=-1)
        _backward(gate, up, output_grad, gate_grad, up_grad)
        return x_grad, None, None


class _SwigluPackedFp8(torch.autograd.Function):
    """_SwigluPacked that keeps its input in 8-bit blocks (quantize_fp8 of x as [.., 2, I]) and differentiates at those values."""

    @staticmethod
    @ensure_contiguous
    def forward(ctx, x: torch.Tensor) -> torch.Tensor:
        half = x.size(-1) // 2
        output = x.new_empty(*x.shape[:-1], half)
        rows = x.numel() // x.size(-1)
        values = torch.empty(rows, 2, half, dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty(rows, 2, 4 * ceil_divide(half, 512), dtype=scales_dtype(), device=x.device)
        swiglu_fp8_forward_cuda(x.view(rows, 2 * half), output.view(rows, half), values, scales)
        ctx.save_for_backward(values, scales)
        return output

    @staticmethod
    @ensure_contiguous
    def backward(ctx, output_grad: torch.Tensor) -> torch.Tensor:
        values, scales = ctx.saved_tensors
        rows, _, half = values.shape
        x_grad = output_grad.new_empty(*output_grad.shape[:-1], 2 * half)
        swiglu_fp8_backward_cuda(values, scales, output_grad.view(rows, half), x_grad.view(rows, 2 * half))
        return x_grad


def swiglu(
    gate: torch.Tensor,
    up: torch.Tensor,
    *,
    kernel_backend_forward: KernelBackend = KernelBackend.cuda,
    kernel_backend_backward: KernelBackend = KernelBackend.cuda,
) -> torch.Tensor:
    """up * gate * sigmoid(gate) for two tensors of the same shape and dtype (fp32 arithmetic, output in their dtype).
    Both backends must name the HIP kernels (KernelBackend.cuda or .triton)."""
    return _Swiglu.apply(gate, up, kernel_backend_forward, kernel_backend_backward)


def swiglu_packed(
    x: torch.Tensor,
    *,
    kernel_backend_forward: KernelBackend = KernelBackend.triton,
    kernel_backend_backward: KernelBackend = KernelBackend.triton,
) -> torch.Tensor:
    """The same activation for x = [up | gate] along the last dimension (which must be even); the result has half
    that length. The defaults are the reference's (`triton`), served here by the HIP kernels."""
    return _SwigluPacked.apply(x, kernel_backend_forward, kernel_backend_backward)


def swiglu_packed_fp8(
    x: torch.Tensor,
    *,
    kernel_backend_forward: KernelBackend = KernelBackend.cuda,
    kernel_backend_backward: KernelBackend = KernelBackend.cuda,
) -> torch.Tensor:
    """swiglu_packed that keeps x for the backward pass in 8 bits (blocks of 128 along each half, see fma.ops.fp8) instead of as it is: half
    the memory in 16-bit types, a quarter in float32. The result is that of swiglu_packed; the gradient is the activation's at the 8-bit
    values."""
    _require_hip(kernel_backend_forward, kernel_backend_backward)
    _check_packed(x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _SwigluPackedFp8.apply(x)
    return swiglu_packed(x, kernel_backend_forward=kernel_backend_forward, kernel_backend_backward=kernel_backend_backward)
