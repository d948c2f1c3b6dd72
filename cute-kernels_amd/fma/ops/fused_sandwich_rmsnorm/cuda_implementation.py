"""Custom ops over fma_sandwich_rmsnorm_fwd and fma_sandwich_rmsnorm_bwd of libfma_hip.so."""

import torch

from ... import _lib
from ..._ops import hip_op


def _check(x: torch.Tensor, like_x: tuple, post_weight, weight, gate, gate_rows: int, stats) -> tuple[int, int, int]:
    """rows, their length and that of the gate's; every argument is what the kernels take it for"""
    shape, dtype, device = x.shape, x.dtype, x.get_device()
    assert len(shape) >= 1 and shape[-1] > 0 and x.is_contiguous(), "x should have rows of one element at least"
    H = shape[-1]
    B = x.numel() // H
    for t in like_x:
        assert t is None or (t.shape == shape and t.dtype is dtype and t.is_contiguous()), "x and residual should be of one shape and dtype"
        assert t is None or t.get_device() == device, "all tensors should be on one device"
    for name, t in (("post_weight", post_weight), ("weight", weight)):
        assert t is None or (t.shape == shape[-1:] and t.dtype is dtype and t.is_contiguous()), f"{name} should be 1-D, of x's row length and dtype"
        assert t is None or t.get_device() == device, "all tensors should be on one device"
    gate_width = 0
    if gate is not None:
        assert gate.dtype is dtype and gate.is_contiguous(), "gate should have x's dtype"
        gate_width = gate.size(-1) if gate.dim() else 1
        assert gate.numel() == gate_rows * gate_width and gate_width in (1, H) and gate.get_device() == device
    assert stats is None or (stats.shape == (2, B) and stats.dtype is torch.float32 and stats.is_contiguous() and stats.get_device() == device)
    return B, H, gate_width


@hip_op("fused_sandwich_rmsnorm_forward_cuda", mutates_args={"output", "stream", "stats"})
def fused_sandwich_rmsnorm_forward_cuda(
    x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor | None, weight: torch.Tensor | None, gate: torch.Tensor | None,
    output: torch.Tensor, stream: torch.Tensor, stats: torch.Tensor | None, gate_rows: int, eps: float, multiplier: float,
) -> None:  # fmt: skip
    B, H, gate_width = _check(x, (residual, output, stream), post_weight, weight, gate, gate_rows, stats)
    _lib.require_gpu(x)  # (and with it the others)
    if B == 0:
        return
    with _lib.on_device(x.device):
        rc = _lib.load().fma_sandwich_rmsnorm_fwd(
            x.data_ptr(), residual.data_ptr(), _lib.ptr(post_weight), _lib.ptr(weight), _lib.ptr(gate), gate_rows, gate_width,
            output.data_ptr(), stream.data_ptr(), _lib.ptr(stats), B, H, eps, multiplier, _lib.dtype_code(x.dtype),
            _lib.current_stream(x.device),
        )  # fmt: skip
    _lib.check(rc, "fused_sandwich_rmsnorm_forward_cuda")


@hip_op("fused_sandwich_rmsnorm_backward_cuda", mutates_args={"x_grad", "residual_grad", "post_weight_grad", "weight_grad", "gate_grad"})
def fused_sandwich_rmsnorm_backward_cuda(
    x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor | None, weight: torch.Tensor | None, gate: torch.Tensor | None,
    output_grad: torch.Tensor | None, stream_grad: torch.Tensor | None, stats: torch.Tensor, x_grad: torch.Tensor,
    residual_grad: torch.Tensor, post_weight_grad: torch.Tensor | None, weight_grad: torch.Tensor | None, gate_grad: torch.Tensor | None,
    gate_rows: int, multiplier: float,
) -> None:  # fmt: skip
    B, H, gate_width = _check(x, (residual, output_grad, stream_grad, x_grad, residual_grad), post_weight, weight, gate, gate_rows, stats)
    for grad, t in ((post_weight_grad, post_weight), (weight_grad, weight), (gate_grad, gate)):
        assert grad is None or (grad.shape == t.shape and grad.dtype is x.dtype and grad.is_contiguous() and grad.get_device() == x.get_device())
    _lib.require_gpu(x)  # (and with it the others)
    lib = _lib.load()
    with _lib.on_device(x.device):
        nbytes = lib.fma_sandwich_rmsnorm_bwd_workspace_bytes(B, H, gate_rows, gate_width)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        rc = lib.fma_sandwich_rmsnorm_bwd(
            x.data_ptr(), residual.data_ptr(), _lib.ptr(post_weight), _lib.ptr(weight), _lib.ptr(gate), gate_rows, gate_width,
            _lib.ptr(output_grad), _lib.ptr(stream_grad), stats.data_ptr(), x_grad.data_ptr(), residual_grad.data_ptr(), _lib.ptr(gate_grad),
            _lib.ptr(post_weight_grad), _lib.ptr(weight_grad), B, H, multiplier, workspace.data_ptr(), nbytes, _lib.dtype_code(x.dtype),
            _lib.current_stream(x.device),
        )  # fmt: skip
    _lib.check(rc, "fused_sandwich_rmsnorm_backward_cuda")
