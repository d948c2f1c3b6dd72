"""Custom ops over fma_router_loss and fma_router_loss_bwd of libfma_hip.so."""

import torch

from ... import _lib
from ..._ops import hip_op


def _check(logits: torch.Tensor, mask: torch.Tensor | None, table: torch.Tensor) -> tuple[int, int]:
    assert logits.dim() == 2 and logits.is_contiguous()
    (T, E), device = logits.shape, logits.get_device()
    assert mask is None or (mask.dtype is torch.bool and mask.shape == (T,) and mask.is_contiguous())
    assert mask is None or mask.get_device() == device, "mask and router_logits should be on one device"
    assert table.dtype is torch.float32 and table.shape == (E + 1,) and table.is_contiguous() and table.get_device() == device
    return T, E


@hip_op("router_loss_cuda", mutates_args={"balance", "z", "counts", "table"})
def router_loss_cuda(
    logits: torch.Tensor, mask: torch.Tensor | None, top_k: int, balance: torch.Tensor, z: torch.Tensor, counts: torch.Tensor,
    table: torch.Tensor,
) -> None:  # fmt: skip
    T, E = _check(logits, mask, table)
    _lib.require_gpu(logits)  # (and with it the others)
    assert balance.dtype is z.dtype is torch.float32 and balance.numel() == z.numel() == 1
    assert counts.dtype is torch.uint32 and counts.shape == (E,) and counts.is_contiguous()
    assert balance.get_device() == z.get_device() == counts.get_device() == logits.get_device()
    lib = _lib.load()
    with _lib.on_device(logits.device):
        nbytes = lib.fma_router_loss_workspace_bytes(T, E)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=logits.device)
        rc = lib.fma_router_loss(
            logits.data_ptr(), _lib.ptr(mask), T, E, top_k, balance.data_ptr(), z.data_ptr(), counts.data_ptr(), table.data_ptr(),
            workspace.data_ptr(), nbytes, _lib.dtype_code(logits.dtype), _lib.current_stream(logits.device),
        )  # fmt: skip
    _lib.check(rc, "router_loss_cuda")


@hip_op("router_loss_backward_cuda", mutates_args={"logits_grad"})
def router_loss_backward_cuda(
    logits: torch.Tensor, mask: torch.Tensor | None, table: torch.Tensor, balance_grad: torch.Tensor | None, z_grad: torch.Tensor | None,
    logits_grad: torch.Tensor,
) -> None:  # fmt: skip
    T, E = _check(logits, mask, table)
    _lib.require_gpu(logits)  # (and with it the others)
    assert logits_grad.shape == logits.shape and logits_grad.dtype is logits.dtype and logits_grad.is_contiguous()
    assert logits_grad.get_device() == logits.get_device()
    for t in (balance_grad, z_grad):
        assert t is None or (t.dtype is torch.float32 and t.numel() == 1 and t.get_device() == logits.get_device())
    with _lib.on_device(logits.device):
        rc = _lib.load().fma_router_loss_bwd(
            logits.data_ptr(), _lib.ptr(mask), T, E, table.data_ptr(), _lib.ptr(balance_grad), _lib.ptr(z_grad), logits_grad.data_ptr(),
            _lib.dtype_code(logits.dtype), _lib.current_stream(logits.device),
        )  # fmt: skip
    _lib.check(rc, "router_loss_backward_cuda")
