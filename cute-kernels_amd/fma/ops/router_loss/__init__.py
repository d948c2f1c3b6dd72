"""`router_loss`: the losses that keep a router even and its logits small, with the tokens of every expert, from the router's logits. The
reference has no counterpart; its layer returns the logits for the caller's own (fma/modules/moe/__init__.py:162-189)."""

import torch
from torch.autograd.function import once_differentiable

from ...kernel_backend import KernelBackend, is_hip_kernel_backend
from .cuda_implementation import router_loss_backward_cuda, router_loss_cuda

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
MAX_EXPERTS = 1024


class _RouterLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, top_k: int, mask: torch.Tensor | None) -> tuple[torch.Tensor, ...]:
        E, device = logits.size(1), logits.device
        balance, z = [torch.empty((), dtype=torch.float32, device=device) for _ in range(2)]
        counts = torch.empty(E, dtype=torch.uint32, device=device)
        table = torch.empty(E + 1, dtype=torch.float32, device=device)  # what the backward needs to know of all tokens
        router_loss_cuda(logits, mask, top_k, balance, z, counts, table)
        ctx.save_for_backward(logits, mask, table)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return balance, z, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, balance_grad: torch.Tensor | None, z_grad: torch.Tensor | None, _) -> tuple[torch.Tensor | None, ...]:
        if balance_grad is None and z_grad is None:
            return None, None, None
        logits, mask, table = ctx.saved_tensors
        logits_grad = torch.empty_like(logits)
        router_loss_backward_cuda(logits, mask, table, balance_grad, z_grad, logits_grad)
        return logits_grad, None, None


def router_loss(
    router_logits: torch.Tensor,
    num_experts_per_tok: int,
    mask: torch.Tensor | None = None,
    kernel_backend: KernelBackend = KernelBackend.triton,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Returns (balance loss, z loss, tokens per expert) of router_logits [.., E], float32, float16 or bfloat16, E <= 1024.

    With p = softmax(logits) per token, f_e the share of all choices that fall on expert e (a token chooses its num_experts_per_tok largest
    logits, the lowest expert first among equal ones) and P_e the mean of p_e over the tokens, the balance loss is E sum_e f_e P_e: 1 if both
    are even. The z loss is the mean of logsumexp(logits)^2. Both are float32 scalars, computed in float32 with sums over tokens joined in
    64 bits, and have gradients by the logits (f counts as a constant; no second derivatives). The tokens per expert are uint32 [E]. A token that
    counts and has no finite softmax (a NaN, +infinity, or nothing but -infinity) makes both losses NaN, and its own gradients.

    mask: bool, one entry per token, False for tokens that do not count (padding): their logits are not looked at, whatever they are, and
    have gradient 0. Its shape is that of the logits without E; to logits [T, E] also any other of T entries, such as [batch, sequence] with
    T = batch * sequence. Without a token that counts both losses are 0. kernel_backend: `triton` (the default) and `cuda` both run the HIP
    kernels; anything else raises ValueError.
    """
    if not is_hip_kernel_backend(kernel_backend):
        raise ValueError(f"unexpected kernel_backend ({kernel_backend})")
    assert router_logits.dtype in _FLOATS, f"router_loss takes float32, float16 and bfloat16, not {router_logits.dtype}"
    assert router_logits.dim() >= 1, "router_logits should have a dimension"
    *tokens, E = router_logits.shape
    assert 1 <= E <= MAX_EXPERTS, f"there should be 1 to {MAX_EXPERTS} experts, not {E}"
    assert 1 <= num_experts_per_tok <= E, f"num_experts_per_tok should be in [1, {E}], not {num_experts_per_tok}"
    logits = (router_logits if len(tokens) == 1 else router_logits.reshape(-1, E)).contiguous()
    if mask is not None:
        assert mask.dtype == torch.bool, "mask should be bool"
        assert mask.shape == tuple(tokens) or (len(tokens) == 1 and mask.numel() == tokens[0]), (
            f"a mask of shape {tuple(mask.shape)} does not fit logits of shape {tuple(router_logits.shape)}"
        )
        mask = mask.reshape(-1).contiguous()
    return _RouterLoss.apply(logits, num_experts_per_tok, mask)
