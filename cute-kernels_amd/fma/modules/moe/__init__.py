"""Mixture-of-Experts layer: the reference's `Experts` and `MoE` modules (fma/modules/moe/__init__.py:17-298) with the
expert computation done by the HIP kernels of libfma_hip.so.

Parameter and buffer names and shapes are the reference's (`gate.weight [E, H]`, `c_fc.weight [E, 2I or I, H]`,
`c_proj.weight [E, H, I]`, uint32 buffers `N_array` / `K_array`), so its state_dicts load unchanged.
"""

from types import MethodType
from typing import Callable

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad

from ...kernel_backend import KernelBackend, is_hip_kernel_backend
from ...ops.swiglu import swiglu_packed
from .fp8_implementation import quantize_expert_weights, requantize_expert_weights, swiglu_experts_fp8
from .cuda_implementation import (
    add_expert_bias,
    build_routing_index,
    combine,
    fp32_router_is_fusable,
    fp32_swiglu_layer,
    fused_router,
    fused_router_with_histogram,
    gathered_swiglu_experts,
    gathered_up_projection_experts,
    MAX_DECODE_EXPERTS,
    MAX_DECODE_ROWS,
    moe_decode,
    swiglu_experts,
    thin_swiglu_experts,
    can_gather_inside_gemm,
    gather_rows,
    grouped_gemm_experts,
    up_projection_swiglu_experts,
)


# The rows of an fp32 layer that runs as three operators, as they are held: tokens, pre-activation and activation in the forward call,
# their gradients in the backward, all at the same time (the general path frees each when the next is there: steps of 512 and 4096
# tokens, hidden 512, I 512, E 16, k 2, peak at 57 and 120 MB, in three operators at 68 and 208 MB). What they save is host time, 350 us
# of a training step: 617 -> 275 us at 8 MB, 734 -> 681 us at 64 MB, 2122 -> 2050 us at 256 MB.
FP32_LAYER_MAX_BYTES = 1 << 28


# (a parameter that nn.Module has accepted is one of these, a tensor subclass, or a fake tensor of a traced layer)
_PLAIN_TENSORS = (torch.Tensor, nn.Parameter)


def _is_traced() -> bool:
    """torch.compile and export, make_fx and fake tensors (whatever else is run under a dispatch mode too), torch.jit.trace"""
    C = torch._C
    return (
        torch.compiler.is_compiling()
        or C._len_torch_dispatch_stack() > 0
        or C._dispatch_tls_is_dispatch_key_included(C.DispatchKey.PreDispatch)
        or C._get_tracing_state() is not None
    )


def _has_global_hooks() -> bool:
    m = nn.modules.module
    return bool(m._global_forward_hooks or m._global_forward_pre_hooks or m._global_backward_hooks or m._global_backward_pre_hooks)


class Experts(nn.Module):
    """The weights (and optional biases) of all experts of one projection: `weight[e]` is expert e's [out, in] matrix."""

    def __init__(
        self, num_experts: int, in_features: int, out_features: int, add_bias: bool = True, std: float | None = None
    ) -> None:
        super().__init__()
        self.num_experts, self.in_features, self.out_features, self.std = num_experts, in_features, out_features, std

        self.weight = nn.Parameter(torch.empty(num_experts, out_features, in_features))
        self.bias = nn.Parameter(torch.empty(num_experts, out_features)) if add_bias else None
        # per-group N and K of the grouped GEMM, kept on the device next to the weights (buffers of the state_dict)
        for name in ("N_array", "K_array"):
            self.register_buffer(name, torch.empty((num_experts,), dtype=torch.uint32))

        self.reset_parameters()

    def cuda_forward(self, input: torch.Tensor, expert_frequency: torch.Tensor) -> torch.Tensor:
        # the reference's cuda_forward (fma/modules/moe/__init__.py:89-92) silently drops the bias; here it is added
        # to the rows of every expert (in the GEMM's epilogue for 16-bit types), which is what its torch_forward
        # computes (:98-105)
        return grouped_gemm_experts(
            x=input, weight=self.weight, M_array=expert_frequency, N_array=self.N_array, K_array=self.K_array,
            bias=self.bias,
        )

    def cuda_forward_swiglu(self, input: torch.Tensor, expert_frequency: torch.Tensor) -> torch.Tensor:
        """up-projection with swiglu_packed fused into the GEMM epilogue: returns [sum(M), out_features / 2]"""
        return up_projection_swiglu_experts(
            x=input, weight=self.weight, M_array=expert_frequency, N_array=self.N_array, K_array=self.K_array,
            bias=self.bias,
        )

    @staticmethod
    def _routing_tensors(
        sorted_scattered_idxs: torch.Tensor, expert_offsets: torch.Tensor
    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """rows per expert (uint32), the routing order and its inverse (int32) from what the reference's callers hold:
        the order of the (token, choice) slots sorted by expert and the inclusive offsets of the experts in it"""
        perm = sorted_scattered_idxs.to(torch.int32).contiguous()
        inverse = torch.empty_like(perm)
        inverse[perm.long()] = torch.arange(perm.numel(), dtype=torch.int32, device=perm.device)
        offsets = expert_offsets.to(torch.int32)
        counts = torch.diff(offsets, prepend=offsets.new_zeros(1))
        return counts.contiguous().view(torch.uint32), perm, inverse

    def up_projection_triton_forward(
        self,
        input: torch.Tensor,
        num_experts_per_token: int | None = None,
        sorted_expert_idxs: torch.Tensor | None = None,
        sorted_scattered_idxs: torch.Tensor | None = None,
        expert_offsets: torch.Tensor | None = None,
    ) -> torch.Tensor:
        """The reference's entry point of this name (fma/modules/moe/__init__.py:40-62: scattered_experts with the tokens
        as input and grouped rows as output), on the HIP kernels: row i of the result is input[sorted_scattered_idxs[i] //
        num_experts_per_token] @ weight[expert of row i]^T, the rows gathered inside the GEMM where its limits allow."""
        assert self.bias is None
        expert_frequency, perm, inverse = self._routing_tensors(sorted_scattered_idxs, expert_offsets)
        if can_gather_inside_gemm(input, self.weight, None):
            return gathered_up_projection_experts(
                input, self.weight, None, perm, inverse, expert_frequency, self.N_array, self.K_array,
                num_experts_per_token, False,
            )  # fmt: skip
        return self.cuda_forward(gather_rows(input, perm, inverse, num_experts_per_token), expert_frequency)

    def down_projection_triton_forward(
        self,
        input: torch.Tensor,
        num_experts_per_token: int | None = None,
        sorted_expert_idxs: torch.Tensor | None = None,
        sorted_scattered_idxs: torch.Tensor | None = None,
        expert_offsets: torch.Tensor | None = None,
        gates: torch.Tensor | None = None,
    ) -> torch.Tensor:
        """The reference's entry point of this name (fma/modules/moe/__init__.py:64-87: scattered_experts with grouped rows
        as input), on the HIP kernels: the projection of the grouped rows, returned per (token, choice) slot, or, with
        `gates` [T, k], as the gate-weighted sum over every token's k rows."""
        assert self.bias is None
        expert_frequency, perm, inverse = self._routing_tensors(sorted_scattered_idxs, expert_offsets)
        output = self.cuda_forward(input, expert_frequency)
        if gates is None:
            # out[slot] = output[row of slot]: the row movement of gather_rows with the two index arrays exchanged
            return gather_rows(output, inverse, perm, 1)
        return combine(output, gates, inverse)

    def extra_repr(self) -> str:
        return f"num_experts={self.num_experts}, in_features={self.in_features}, out_features={self.out_features}"

    @torch.no_grad()
    def reset_parameters(self) -> None:
        # N(0, std) weights, zero biases (fma/modules/moe/__init__.py:112-121), and the two size buffers
        nn.init.normal_(self.weight, mean=0, std=self.std)
        if getattr(self, "bias", None) is not None:
            self.bias.zero_()
        self.N_array.fill_(self.out_features)
        self.K_array.fill_(self.in_features)


def _is_swiglu_packed(activation_function: Callable) -> bool:
    fn = getattr(activation_function, "func", activation_function)  # functools.partial(swiglu_packed, ...)
    return fn is swiglu_packed


class MoE(nn.Module):
    # (of the class as well: a pickled layer from before they existed has none of its own)
    fp8_experts = False
    _fp8_weights: tuple | None = None

    def __init__(
        self,
        num_experts: int,
        num_experts_per_tok: int,
        hidden_size: int,
        intermediate_size: int,
        activation_function: Callable,
        is_glu: bool,
        add_bias: bool,
        std: float,
    ) -> None:
        super().__init__()

        self.num_experts = num_experts
        self.top_k = num_experts_per_tok

        self.hidden_size = hidden_size
        self.intermediate_size = intermediate_size

        self.gate = nn.Linear(in_features=self.hidden_size, out_features=num_experts, bias=False)
        # gate GEMM, top-k and softmax in one kernel wherever that kernel applies (16-bit activations on the GPU)
        self.fuse_router = True

        self.c_fc = Experts(
            num_experts=num_experts,
            in_features=self.hidden_size,
            out_features=2 * self.intermediate_size if is_glu else self.intermediate_size,
            add_bias=add_bias,
            std=std,
        )

        # None: decided per call (see _gathers_inside_gemm); True / False: always / never
        self.gather_in_gemm: bool | None = None
        # the activation's backward inside the second projection's input-gradient GEMM (see _runs_swiglu_experts_as_one_node)
        self.fuse_swiglu_backward = True

        # The experts' products in 8 bits (swiglu_experts_fp8): a SwiGLU layer without biases in a 16-bit type. 16 / 8 bits, us: hidden 2048, I 1408,
        # E 64, k 8, prepared weights, 1 token 34 / 38 (called eagerly 36 / 80), 16 tokens 174 / 124, 4096 tokens 560 / 366; training steps of 8192 and
        # 32768 tokens 3438 / 3471, 12250 / 11835; hidden 4096, I 1536, E 128, k 8, 1 token 64 / 62, 4096 tokens 1398 / 823, a training step
        # of 8192 tokens 7578 / 8436, which keeps 3362 MB instead of 1211 (8-bit copies of the weights among them).
        self.fp8_experts = False
        self._fp8_weights = None  # what quantize_experts() made, and the versions it made it of

        self.act = activation_function
        # swiglu_packed as the activation of a GLU layer is computed inside the up-projection's epilogue (a kernel for
        # rows of whole 16-byte pieces; other sizes run the GEMM's element-wise path and the activation after it)
        self.fuse_swiglu = (
            is_glu
            and _is_swiglu_packed(activation_function)
            and self.hidden_size % 8 == 0
            and self.intermediate_size % 8 == 0
        )

        self.c_proj = Experts(
            num_experts=num_experts,
            in_features=self.intermediate_size,
            out_features=self.hidden_size,
            add_bias=add_bias,
            std=std,
        )

    def forward(
        self, hidden_states: torch.Tensor, kernel_backend: KernelBackend = KernelBackend.triton
    ) -> tuple[torch.Tensor, torch.Tensor]:
        original_shape = hidden_states.shape

        # hidden_states -> (total_q, hidden_size)
        hidden_states = hidden_states.view(-1, self.hidden_size)
        operands = self._decode_operands(hidden_states, kernel_backend)
        if operands is not None:
            hidden_states, router_logits = moe_decode(hidden_states.contiguous(), *operands, self.top_k)
            return hidden_states.view(original_shape), router_logits
        operands = self._fp32_operands(hidden_states, kernel_backend)
        if operands is not None:
            routed = None
            if not fp32_router_is_fusable(hidden_states.size(0), self.num_experts, self.hidden_size, self.top_k):
                routed = self._compute_routing_weights(hidden_states)
            hidden_states, router_logits = fp32_swiglu_layer(hidden_states, *operands, self.top_k, routed)
            return hidden_states.view(original_shape), router_logits

        token_block_histogram = None
        if self._router_is_fusable(hidden_states):
            # the router kernel counts its choices as it makes them; the index build starts from those counts
            router_logits, router_weights, selected_experts, token_block_histogram = fused_router_with_histogram(
                hidden_states, self.gate.weight, self.top_k
            )
        else:
            router_logits, router_weights, selected_experts = self._compute_routing_weights(hidden_states)

        # router_logits -> (total_q, num_experts); router_weights, selected_experts -> (total_q, top_k)
        hidden_states = self._compute_experts(
            hidden_states,
            router_weights,
            selected_experts,
            kernel_backend=kernel_backend,
            token_block_histogram=token_block_histogram,
        )

        hidden_states = hidden_states.view(original_shape)

        return hidden_states, router_logits

    def _router_is_fusable(self, hidden_states: torch.Tensor, gate_weight: torch.Tensor | None = None) -> bool:
        # the last three lines are the size limits of fma_router_topk (32-bit offsets into logits and choices): larger
        # inputs take the library calls below instead of raising
        T = hidden_states.size(0)
        return (
            self.fuse_router
            and hidden_states.is_cuda
            and hidden_states.dtype in (torch.bfloat16, torch.float16)
            and (self.gate.weight if gate_weight is None else gate_weight).dtype == hidden_states.dtype
            and self.hidden_size % 8 == 0
            and self.num_experts <= 1024
            and self.top_k <= 64
            and self.hidden_size <= (1 << 24)
            and T * self.num_experts <= 2**31 - 1
            and T * self.top_k <= 2**31 - 1
        )

    def _compute_routing_weights(self, hidden_states: torch.Tensor) -> tuple[torch.Tensor]:
        if self._router_is_fusable(hidden_states):
            # same three results; selected_experts comes back as int32, sorted by descending logit
            return fused_router(hidden_states, self.gate.weight, self.top_k)

        router_logits = self.gate(hidden_states)
        router_weights, selected_experts = self._get_topk(router_logits)

        # softmax over the k kept logits, in fp32
        router_weights = F.softmax(router_weights.float(), dim=-1)
        router_weights = router_weights.type_as(hidden_states)

        return router_logits, router_weights, selected_experts

    def _compute_experts(
        self,
        hidden_states: torch.Tensor,
        router_weights: torch.Tensor,
        selected_experts: torch.Tensor,
        kernel_backend: KernelBackend,
        token_block_histogram: torch.Tensor | None = None,
    ) -> torch.Tensor:
        if not is_hip_kernel_backend(kernel_backend):
            raise ValueError(f"unexpected kernel_backend ({kernel_backend})")

        if self.fp8_experts:
            return self._compute_experts_fp8(hidden_states, router_weights, selected_experts)

        # counts, offsets and the stable expert-major order of the (token, choice) slots, with its inverse
        expert_frequency, expert_offsets, sorted_scattered_idxs, _, inverse = build_routing_index(
            selected_experts, self.num_experts, token_block_histogram
        )

        if self._runs_thin_experts(hidden_states, selected_experts.numel()):
            hidden_states = thin_swiglu_experts(
                hidden_states, self.c_fc.weight, self.c_fc.bias, self.c_proj.weight, self.c_proj.bias,
                sorted_scattered_idxs, expert_frequency, expert_offsets, self.top_k,
            )  # fmt: skip
            return combine(hidden_states, router_weights, inverse)

        if self._gathers_inside_gemm(hidden_states):
            # the first projection (and its weight gradient) reads its rows x[slot // top_k] through the routing order: no
            # grouped copy of x
            if self._runs_swiglu_experts_as_one_node(hidden_states):
                hidden_states = gathered_swiglu_experts(
                    hidden_states, self.c_fc.weight, self.c_fc.bias, self.c_proj.weight, self.c_proj.bias,
                    sorted_scattered_idxs, inverse, expert_frequency, self.c_fc.N_array, self.c_fc.K_array,
                    self.c_proj.N_array, self.c_proj.K_array, self.top_k,
                )  # fmt: skip
                return combine(hidden_states, router_weights, inverse)
            fused = self.fuse_swiglu
            hidden_states = gathered_up_projection_experts(
                hidden_states, self.c_fc.weight, self.c_fc.bias, sorted_scattered_idxs, inverse, expert_frequency,
                self.c_fc.N_array, self.c_fc.K_array, self.top_k, fused,
            )  # fmt: skip
            if not fused:
                hidden_states = self.act(hidden_states)
            hidden_states = self.c_proj.cuda_forward(input=hidden_states, expert_frequency=expert_frequency)
            return combine(hidden_states, router_weights, inverse)

        # rows of every expert back to back: x[slot // top_k]
        hidden_states = gather_rows(hidden_states, sorted_scattered_idxs, inverse, self.top_k)

        if self._runs_swiglu_experts_as_one_node(hidden_states):
            # both projections in one autograd node: its backward forms the pre-activation's gradient in one kernel
            hidden_states = swiglu_experts(
                hidden_states, self.c_fc.weight, self.c_fc.bias, self.c_proj.weight, self.c_proj.bias, expert_frequency,
                self.c_fc.N_array, self.c_fc.K_array, self.c_proj.N_array, self.c_proj.K_array,
            )  # fmt: skip
            return combine(hidden_states, router_weights, inverse)

        if self.fuse_swiglu and hidden_states.dtype in (torch.bfloat16, torch.float16):
            hidden_states = self.c_fc.cuda_forward_swiglu(input=hidden_states, expert_frequency=expert_frequency)
        else:
            hidden_states = self.c_fc.cuda_forward(input=hidden_states, expert_frequency=expert_frequency)
            hidden_states = self.act(hidden_states)

        hidden_states = self.c_proj.cuda_forward(input=hidden_states, expert_frequency=expert_frequency)

        # y[t] = sum_j router_weights[t, j] * expert_output[row of slot (t, j)]
        hidden_states = combine(hidden_states, router_weights, inverse)

        return hidden_states

    def quantize_experts(self) -> "MoE":
        """Switches the experts' products to 8 bits (fp8_experts) and lays both projections out in 8 bits once, for calls that no backward
        pass follows: a serving program of more than a token or two at a time (see __init__) calls it after loading the weights, and again
        after changing them. A forward pass on weights that
        have changed since, as far as their version counters tell, quantises them in the call, as one without this call does; changes that
        no counter sees (through .data, or by a replayed graph) need the call again. A compiled layer quantises in the call. Called again, it
        writes to the same memory, so that a graph captured before serves the new weights (unless they are on another device since)."""
        if any(t.is_inference() for t in (self.c_fc.weight, self.c_proj.weight)):
            raise ValueError("quantize_experts: parameters that were made in inference mode do not tell when they change")
        self._check_fp8_experts(self.c_fc.weight.dtype)
        with torch.inference_mode(False), torch.no_grad():  # (a later call writes to what is made here, in whatever mode)
            weights, blocks = (self.c_fc.weight, self.c_proj.weight), self._fp8_weights and self._fp8_weights[1]
            if blocks and all(b.values.device == w.device for b, w in zip(blocks, weights)):
                requantize_expert_weights(*weights, *blocks)
            else:
                blocks = quantize_expert_weights(*weights)
            self._fp8_weights = (self._weight_versions(), blocks)
        self.fp8_experts = True
        return self

    def _weight_versions(self) -> tuple:
        # (module.to() puts other memory behind a parameter without advancing its version)
        return tuple((t, t._version, t.data_ptr(), t.dtype) for t in (self.c_fc.weight, self.c_proj.weight))

    def _check_fp8_experts(self, dtype: torch.dtype) -> None:
        if not (self.c_fc.out_features == 2 * self.intermediate_size and _is_swiglu_packed(self.act)):
            raise ValueError("fp8_experts: the layer's activation should be swiglu_packed")
        if self.c_fc.bias is not None or self.c_proj.bias is not None:
            raise ValueError("fp8_experts: a layer with biases has no 8-bit path")
        if dtype not in (torch.bfloat16, torch.float16) or not self.c_fc.weight.dtype == self.c_proj.weight.dtype == dtype:
            raise ValueError("fp8_experts: tokens and weights should both be bfloat16 or float16")
        if self.hidden_size % 16 != 0 or self.intermediate_size % 16 != 0:
            raise ValueError("fp8_experts: hidden and intermediate size should be multiples of 16")

    def _compute_experts_fp8(
        self, hidden_states: torch.Tensor, router_weights: torch.Tensor, selected_experts: torch.Tensor
    ) -> torch.Tensor:
        self._check_fp8_experts(hidden_states.dtype)
        weights = self.c_fc.weight, self.c_proj.weight
        if self._fp8_weights is not None and not torch.is_grad_enabled() and not torch.compiler.is_compiling():
            made_of, blocks = self._fp8_weights
            if all(a[0] is b[0] and a[1:] == b[1:] for a, b in zip(made_of, self._weight_versions())):
                weights = blocks
        return swiglu_experts_fp8(hidden_states, router_weights, selected_experts, *weights)

    def _decode_operands(self, hidden_states: torch.Tensor, kernel_backend: KernelBackend) -> tuple | None:
        """The weights and biases of the layer if the whole forward pass is one native call: no backward, up to 32 rows per expert
        on average (the line of _runs_thin_experts, whose kernel it runs) and up to 1024 (token, choice) slots (one workgroup sorts
        them). (Each parameter is looked up once: a look-up in a module takes 0.3 us of host time, and a token is 42 us.)"""
        rows = hidden_states.size(0) * self.top_k
        if not (
            0 < rows <= MAX_DECODE_ROWS
            and self.num_experts <= MAX_DECODE_EXPERTS
            and not torch.is_grad_enabled()
            and hidden_states.is_cuda
            and hidden_states.dtype in (torch.bfloat16, torch.float16)
            and self.fuse_router
            and self.fuse_swiglu
            and self.gather_in_gemm is not False
            and not self.fp8_experts
        ):
            return None
        parameters, gate_weight = self._expert_parameters(), self.gate.weight
        if not (
            self._runs_thin_experts(hidden_states, rows, parameters)
            and self._router_is_fusable(hidden_states, gate_weight)
            and is_hip_kernel_backend(kernel_backend)
            # a subclass's own is called, and so is one that was put on the instance
            and isinstance(self._compute_experts, MethodType)
            and self._compute_experts.__func__ is MoE._compute_experts
            and self._compute_experts.__self__ is self
        ):
            return None
        for t in parameters:
            if t is not None and not t.is_contiguous():
                return None
        return (gate_weight, *parameters) if gate_weight.is_contiguous() else None

    def _fp32_operands(self, hidden_states: torch.Tensor, kernel_backend: KernelBackend) -> tuple | None:
        """The weights and sizes of the layer if it is one in fp32 that runs as three operators: a SwiGLU layer without biases, made
        of this file's own parts and the library's nn.Linear, with nothing put in their way (hooks, methods of a subclass or an
        instance, autocast, transforms, tracing). Anything else takes the general path."""
        if hidden_states.dtype is not torch.float32 or not hidden_states.is_cuda or _is_traced():
            return None
        gate, c_fc, c_proj = self.gate, self.c_fc, self.c_proj
        T = hidden_states.size(0)
        if not (
            T > 0
            and type(self) is MoE
            and type(gate) is nn.Linear
            and type(c_fc) is Experts
            and type(c_proj) is Experts
            and self.act is swiglu_packed
            and self.fuse_router
            and self.fuse_swiglu
            and self.fuse_swiglu_backward
            and not self.fp8_experts
            and self.num_experts <= 1024
            and self.top_k <= 64
            and self.hidden_size <= (1 << 24)
            and (self.hidden_size | self.intermediate_size) % 8 == 0  # (the general path refuses others)
            and T * max(self.num_experts, self.top_k) <= 2**31 - 1
            and T * self.top_k * (self.hidden_size + 3 * self.intermediate_size) * 4 <= FP32_LAYER_MAX_BYTES
            and is_hip_kernel_backend(kernel_backend)
            and not torch.is_autocast_enabled("cuda")
            and forward_ad._current_level < 0
            and not torch._C._are_functorch_transforms_active()
        ):
            return None
        own = self.__dict__
        if "_compute_experts" in own or "_compute_routing_weights" in own or "_get_topk" in own or "_router_is_fusable" in own:
            return None
        if "forward" in gate.__dict__ or "cuda_forward" in c_fc.__dict__ or "cuda_forward" in c_proj.__dict__:
            return None
        if gate._forward_hooks or gate._forward_pre_hooks or gate._backward_hooks or gate._backward_pre_hooks or _has_global_hooks():
            return None
        gate_weight, weight1, weight2 = gate.weight, c_fc.weight, c_proj.weight
        for t in (hidden_states, gate_weight, weight1, weight2):
            if type(t) not in _PLAIN_TENSORS:
                return None
        if not (
            gate.bias is None
            and c_fc.bias is None
            and c_proj.bias is None
            and gate_weight.dtype is weight1.dtype is weight2.dtype is torch.float32
            and gate_weight.shape == (self.num_experts, self.hidden_size)
            and (hidden_states.data_ptr() | gate_weight.data_ptr()) % 16 == 0
        ):
            return None
        return gate_weight, weight1, weight2, c_fc.N_array, c_fc.K_array, c_proj.N_array, c_proj.K_array

    def _expert_parameters(self) -> tuple:
        c_fc, c_proj = self.c_fc, self.c_proj
        return c_fc.weight, c_fc.bias, c_proj.weight, c_proj.bias

    def _runs_thin_experts(self, hidden_states: torch.Tensor, rows: int, parameters: tuple | None = None) -> bool:
        """Whether the two projections of a forward pass without a backward run on the kernel for a few rows per expert, which
        streams the weights past them: up to 32 rows per expert on average. Both projections together, that kernel against the
        tile kernel: 16 rows (64 tokens, hidden 4096, I 14336, E 8, k 2) 471 against 547 us, 32 rows 501 against 553 us, 48
        rows 540 against 558 us, 64 rows 834 against 788 us; E 64 (hidden 2048, I 1408, k 8) at 32 rows 235 against 258 us,
        at 64 rows 354 against 290 us. (48 rows on average already have experts beyond the 64 rows of one pass.)"""
        if torch.is_grad_enabled() or not self.fuse_swiglu or self.gather_in_gemm is False:
            return False
        parameters = parameters or self._expert_parameters()
        return (
            # no_grad leaves forward mode and functorch's transforms on, which the autograd nodes of the general path refuse
            forward_ad._current_level < 0
            and not torch._C._are_functorch_transforms_active()
            and rows <= 32 * min(self.num_experts, rows)
            # the general path is one node too: with the switch off it calls the methods of the two Experts modules
            and self._runs_swiglu_experts_as_one_node(hidden_states, parameters)
            and can_gather_inside_gemm(hidden_states, *parameters[:2])
            and self.intermediate_size < (1 << 21)
        )

    def _runs_swiglu_experts_as_one_node(self, hidden_states: torch.Tensor, parameters: tuple | None = None) -> bool:
        """fuse_swiglu_backward: with the fused SwiGLU up-projection, run the second projection in the same autograd node
        so that its input gradient and the activation's backward are one kernel (16-bit types; the sizes that kernel takes)"""
        if not (self.fuse_swiglu and self.fuse_swiglu_backward and hidden_states.dtype in (torch.bfloat16, torch.float16)):
            return False
        dtype = hidden_states.dtype
        weight1, bias1, weight2, bias2 = parameters or self._expert_parameters()
        return (
            weight1.dtype == weight2.dtype == dtype
            and (bias1 is None or bias1.dtype == dtype)
            and (bias2 is None or bias2.dtype == dtype)
            and self.intermediate_size < (1 << 22)
            and self.hidden_size < (1 << 21)
        )

    def _gathers_inside_gemm(self, hidden_states: torch.Tensor) -> bool:
        """Whether the first projection (forward and weight gradient) gathers its rows itself instead of reading a grouped
        copy of the tokens. gather_in_gemm None: when the projection is narrow enough for the saved row-movement pass to
        outweigh the slower operand fetch of scattered rows; True / False force it.

        Whole passes, gathered against copied: without a backward -9 to -1 % up to 5760 columns (512 to 8192 tokens), -3 to +1 %
        from 7168 to 16384, up to +1.4 % at 28672. With one, -3 to +0.8 % from 256 rows per expert on; with fewer the copy would be
        faster: at 128 rows by 2 to 6 %, at 64 and 32 by 4 to 10 % (hidden 4096, I 1536, E 128, 1021 tokens 3399 us gathered, 3091
        copied), since a tile of the weight gradient with two K steps or fewer starts cold in the gathered kernel. The layer
        gathers there too: it then keeps the tokens for the backward and not T * top_k rows of them."""
        if self.gather_in_gemm is False or not can_gather_inside_gemm(hidden_states, self.c_fc.weight, self.c_fc.bias):
            return False
        if self.gather_in_gemm:
            return True
        return self.c_fc.out_features <= 6144

    def _get_topk(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        if self.top_k == 1:
            x, indices = x.max(dim=-1, keepdim=True)
        else:
            x, indices = x.topk(self.top_k, dim=-1)

        return x, indices
