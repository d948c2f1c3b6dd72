"""Calls of fma_grad_norm, fma_scale_grads (and its form for 64-bit norms) and fma_clip_grad_norm of libfma_hip.so. They take lists of tensors
that may be a few hundred, and are no operators of the dispatcher, which would look at each of them twice more."""

from array import array

import torch
from torch._C import _increment_version

from ... import _lib

_TENSORS = {torch.Tensor, torch.nn.Parameter}
_STRIDED = {torch.strided}


def _is_dense(t: torch.Tensor) -> bool:
    """whether the elements fill one piece of memory, in whatever order"""
    if t.is_contiguous():
        return True
    return t.permute(sorted(range(t.dim()), key=t.stride, reverse=True)).is_contiguous()


class _Table:
    """What the library needs to know of the tensors. Those with gaps between their elements come as copies; `copied` says which of what.
    (One look at all tensors for each of their properties: a loop over the tensors with all of them inside takes twice as long.)"""

    def __init__(self, tensors: list[torch.Tensor], written: bool) -> None:
        if not {type(t) for t in tensors} <= _TENSORS or {t.layout for t in tensors} != _STRIDED:
            kinds = ", ".join(sorted({f"{type(t).__name__} of layout {t.layout}" for t in tensors}))
            raise TypeError(f"dense tensors are taken, not {kinds}")
        self.device = tensors[0].device
        if len({t.get_device() for t in tensors}) > 1:
            raise RuntimeError("all tensors should be on one device: got " + ", ".join(sorted({str(t.device) for t in tensors})))
        _lib.require_gpu(tensors[0])
        self.copied, self.views = [], set()
        if not all([t.is_contiguous() for t in tensors]):
            tensors = [self._dense(t, written) for t in tensors]
        self.tensors = tensors  # (holds the copies)
        self._pointers = array("Q", [t.data_ptr() for t in tensors])
        self._sizes = array("q", [t.numel() for t in tensors])
        codes = {d: _lib.dtype_code(d) for d in {t.dtype for t in tensors}}
        if len(codes) == 1:
            self._dtypes = array("i", codes.values()) * len(tensors)
        else:
            self._dtypes = array("i", [codes[t.dtype] for t in tensors])
        self.arguments = *(a.buffer_info()[0] for a in (self._pointers, self._sizes, self._dtypes)), len(tensors)

    def _dense(self, t: torch.Tensor, written: bool) -> torch.Tensor:
        if _is_dense(t):
            return t
        if written and torch._debug_has_internal_overlap(t) == 1:
            raise RuntimeError("a gradient has elements that share memory: make it contiguous first")
        if written:
            view = t.data_ptr(), t.shape, t.stride()
            if view in self.views:
                raise RuntimeError("two gradients share memory")
            self.views.add(view)
        copy = t.contiguous()
        self.copied.append((t, copy))
        return copy


@torch.no_grad()
def grad_norm_cuda(tensors: list[torch.Tensor], infinity: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """the norm, and the workspace, whose first 8 bytes are the norm in 64 bits"""
    table, lib = _Table(tensors, False), _lib.load()
    with _lib.on_device(table.device):
        norm = torch.empty((), dtype=torch.float32, device=table.device)
        nbytes = lib.fma_grad_norm_workspace_bytes(len(tensors))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=table.device)
        rc = lib.fma_grad_norm(
            *table.arguments, infinity, norm.data_ptr(), workspace.data_ptr(), nbytes, _lib.current_stream(table.device)
        )
    _lib.check(rc, "get_total_norm")
    return norm, workspace


def _written(table: _Table, grads: list[torch.Tensor]) -> None:
    for t, copy in table.copied:
        t.copy_(copy)
    _increment_version(grads)


@torch.no_grad()
def scale_grads_cuda(grads: list[torch.Tensor], max_norm: float, norm: torch.Tensor) -> None:
    if not grads:
        return
    table, lib = _Table(grads, True), _lib.load()
    assert norm.numel() == 1, "total_norm should be a scalar"
    # (a norm of any other type than float32 goes as 64 bits)
    dtype, scale = (torch.float32, lib.fma_scale_grads) if norm.dtype is torch.float32 else (torch.float64, lib.fma_scale_grads_norm64)
    norm = norm.to(device=table.device, dtype=dtype)
    with _lib.on_device(table.device):
        rc = scale(*table.arguments, norm.data_ptr(), max_norm, _lib.current_stream(table.device))
    _lib.check(rc, "clip_grads_with_norm_")
    _written(table, grads)


@torch.no_grad()
def clip_grad_norm_cuda(grads: list[torch.Tensor], infinity: bool, max_norm: float) -> torch.Tensor:
    if not grads:
        return torch.tensor(0.0)
    table, lib = _Table(grads, True), _lib.load()
    with _lib.on_device(table.device):
        norm = torch.empty((), dtype=torch.float32, device=table.device)
        nbytes = lib.fma_grad_norm_workspace_bytes(len(grads))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=table.device)
        rc = lib.fma_clip_grad_norm(
            *table.arguments, infinity, max_norm, norm.data_ptr(), workspace.data_ptr(), nbytes, _lib.current_stream(table.device)
        )
    _lib.check(rc, "clip_grad_norm_")
    _written(table, grads)
    return norm
