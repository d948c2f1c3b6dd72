"""The norm of many tensors together and clipping gradients to it, with the names and arguments of torch.nn.utils:

    clip_grad_norm_(parameters, max_norm)                  both, in two passes over the gradients
    get_total_norm(tensors)                                the norm alone
    clip_grads_with_norm_(parameters, max_norm, norm)      scaling by a norm that is known, e.g. one that was reduced over ranks

Norms are those of the elements on this device, as one long vector: 2-norm or largest magnitude. The squares are added in 64 bits and the
result is float32, whatever the tensors' types (which may differ). The reference has no counterpart.

What differs from torch.nn.utils: other norms than 2 and infinity raise ValueError, other types and subclasses of tensors TypeError, tensors on
several devices RuntimeError, and so do most gradients to be scaled that share memory (clip_grad_norm_ says which); a norm has float32, not
the gradients' type; a parameter that comes twice has one gradient; the tensors always go together, so `foreach` is taken and changes nothing."""

import math
from typing import Iterable

import torch

from .cuda_implementation import clip_grad_norm_cuda, grad_norm_cuda, scale_grads_cuda


def _gradients(parameters: torch.Tensor | Iterable[torch.Tensor]) -> list[torch.Tensor]:
    """a parameter that comes twice (a tied one) has one gradient"""
    if isinstance(parameters, torch.Tensor):
        parameters = (parameters,)
    return [grad for grad in [p.grad for p in {id(p): p for p in parameters}.values()] if grad is not None]


def _is_infinity_norm(norm_type: float) -> bool:
    norm_type = float(norm_type)
    if norm_type != 2.0 and norm_type != math.inf:
        raise ValueError(f"norm_type should be 2 or inf, not {norm_type}")
    return norm_type == math.inf


def _check_bound(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm should not be negative, got {max_norm}")
    return max_norm


def _require_finite(norm: torch.Tensor) -> None:
    if not math.isfinite(norm.item()):
        raise RuntimeError("the total norm is not finite, so nothing was clipped; error_if_nonfinite=False clips by it all the same")


def get_total_norm(
    tensors: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0, error_if_nonfinite: bool = False, foreach: bool | None = None
) -> torch.Tensor:
    """The norm (norm_type 2 or inf) of all elements of the tensors (float32, float16, bfloat16, on one GPU): a float32 scalar there. A tensor
    that comes twice counts twice. error_if_nonfinite waits for the result and raises RuntimeError unless it is finite as float32."""
    infinity = _is_infinity_norm(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    norm, _ = grad_norm_cuda(tensors, infinity)
    if error_if_nonfinite:
        _require_finite(norm)
    return norm


def clip_grads_with_norm_(
    parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, total_norm: torch.Tensor, foreach: bool | None = None
) -> None:
    """Multiplies the parameters' gradients, in place, by min(1, max_norm / (total_norm + 1e-6)), which is formed in 64 bits from the total_norm
    as it is given. With a factor of one they are not touched. A total_norm that is itself an element of such a gradient is refused
    (RuntimeError) if the gradient is dense."""
    scale_grads_cuda(_gradients(parameters), _check_bound(max_norm), total_norm)


def clip_grad_norm_(
    parameters: torch.Tensor | Iterable[torch.Tensor],
    max_norm: float,
    norm_type: float = 2.0,
    error_if_nonfinite: bool = False,
    foreach: bool | None = None,
) -> torch.Tensor:
    """Clips the gradients of the parameters to max_norm in place and returns their norm from before: get_total_norm and
    clip_grads_with_norm_ as one call. Parameters without a gradient are passed over. Gradients that share memory are refused (RuntimeError)
    if they are dense or one strided view; different views that overlap are scaled once, and count twice in the norm.
    The gradients are scaled by the norm in 64 bits; one past float32's range comes back as infinity. With error_if_nonfinite a norm that is
    infinite or NaN in 64 bits raises RuntimeError before anything is scaled; the call waits for it and changes no bit otherwise. Not
    traced: a compiled function that calls it breaks its graph here."""
    infinity, max_norm = _is_infinity_norm(norm_type), _check_bound(max_norm)
    grads = _gradients(parameters)
    if error_if_nonfinite and grads:
        norm, workspace = grad_norm_cuda(grads, infinity)
        norm64 = workspace[:8].view(torch.float64)  # what the call without the check scales by, too
        _require_finite(norm64)
        scale_grads_cuda(grads, max_norm, norm64)
        return norm
    return clip_grad_norm_cuda(grads, infinity, max_norm)
