"""Tensors in 8 bits, in blocks of 128, and products of them:

    quantize_fp8(x) / dequantize_fp8(blocks)   to the format and back
    grouped_gemm_fp8(A, B, M_array)            D_e = A_e B_e^T of operands that are in 8 bits already
    grouped_linear_fp8(x, weight, M_array)     y_e = x_e W_e^T from 16-bit tensors, with gradients

A block is 128 neighbouring elements of a row (activations), or 128 x 128 elements of a matrix (weights). Its values are e4m3, its scale is
a power of two (e8m0): the smallest that brings the block's largest magnitude to 448 or less, 2^-126 at the least. value = x / scale,
rounded to nearest even. A block that holds an infinity or a NaN is NaN throughout. The reference has no counterpart."""

from typing import NamedTuple

import torch

from ...math import ceil_divide
from ...utils import ensure_contiguous
from .cuda_implementation import dequantize_fp8_cuda, grouped_gemm_fp8_cuda, quantize_fp8_cuda

BLOCK_SIZE = 128
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class Fp8Blocks(NamedTuple):
    """values: float8_e4m3fn [.., N, K]. scales: float8_e8m0fnu [.., N, P], one per 128 elements of a row, or [.., ceil(N / 128), P], one
    per 128 x 128 elements; P is ceil(K / 128) rounded up to a multiple of four, the entries past ceil(K / 128) are one."""

    values: torch.Tensor
    scales: torch.Tensor


def scale_columns(K: int) -> int:
    return 4 * ceil_divide(K, 4 * BLOCK_SIZE)


def _empty_blocks(shape: tuple[int, ...], block_rows: int, device: torch.device) -> Fp8Blocks:
    *batch, N, K = shape
    return Fp8Blocks(
        torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
        torch.empty(*batch, ceil_divide(N, block_rows), scale_columns(K), dtype=torch.float8_e8m0fnu, device=device),
    )


@torch.no_grad()
@ensure_contiguous
def quantize_fp8(
    x: torch.Tensor, block_rows: int = 1, transposed: bool = False
) -> Fp8Blocks | tuple[Fp8Blocks, Fp8Blocks]:
    """x [.., K] (at least 2-dimensional with block_rows 128; float32, float16 or bfloat16) in 8-bit blocks of block_rows (1 or 128) x 128
    elements. transposed (block_rows 128 only): returns the blocks and those of x.transpose(-1, -2), which are the same blocks."""
    assert block_rows in (1, BLOCK_SIZE), "blocks have 1 or 128 rows"
    assert x.dtype in _FLOATS, f"quantize_fp8 takes float32, float16 and bfloat16, not {x.dtype}"
    assert not transposed or block_rows == BLOCK_SIZE, "a transposed copy exists of 128 x 128 blocks only"
    assert x.dim() >= (1 if block_rows == 1 else 2), "x has too few dimensions"
    assert x.size(-1) > 0, "rows must not be empty"
    shape = tuple(x.shape) if x.dim() > 1 else (1, x.size(0))
    assert not transposed or shape[-2] > 0, "columns must not be empty"
    blocks = _empty_blocks(shape, block_rows, x.device)
    other = _empty_blocks((*shape[:-2], shape[-1], shape[-2]), block_rows, x.device) if transposed else None
    quantize_fp8_cuda(x.view(shape), *blocks, *(other or (None, None)), block_rows)
    if x.dim() == 1:
        return Fp8Blocks(blocks.values[0], blocks.scales[0])
    return blocks if other is None else (blocks, other)


def block_rows_of(blocks: Fp8Blocks) -> int:
    """1 or 128, from the shapes; raises if they do not fit each other"""
    values, scales = blocks
    assert values.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu, "values in e4m3, scales in e8m0"
    assert values.dim() == scales.dim() >= 2, "values and scales should have the same number of dimensions, two at least"
    *batch, N, K = values.shape
    for block_rows in (1, BLOCK_SIZE):
        if K > 0 and scales.shape == (*batch, ceil_divide(N, block_rows), scale_columns(K)):
            return block_rows
    raise AssertionError(f"scales of shape {tuple(scales.shape)} do not fit values of shape {tuple(values.shape)}")


@torch.no_grad()
@ensure_contiguous
def dequantize_fp8(blocks: Fp8Blocks, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that the blocks stand for, rounded to dtype (exact in float32 and bfloat16)."""
    assert dtype in _FLOATS, f"dequantize_fp8 gives float32, float16 and bfloat16, not {dtype}"
    one_row = blocks[0].dim() == 1
    if one_row:
        blocks = Fp8Blocks(blocks[0][None], blocks[1][None])
    block_rows = block_rows_of(blocks)
    output = torch.empty(blocks[0].shape, dtype=dtype, device=blocks[0].device)
    dequantize_fp8_cuda(*blocks, output, block_rows)
    return output[0] if one_row else output


def _check_sizes(M_array: torch.Tensor | None, E: int) -> None:
    if M_array is not None:
        assert M_array.dtype == torch.uint32 and M_array.shape == (E,), "M_array should be uint32 with one entry per group"


@torch.no_grad()
@ensure_contiguous
def grouped_gemm_fp8(
    A: Fp8Blocks, B: Fp8Blocks, M_array: torch.Tensor | None = None, output_dtype: torch.dtype = torch.bfloat16
) -> torch.Tensor:
    """D_e = A_e B_e^T for every group e, fp32 sums, rounded once to output_dtype (bfloat16, float16 or float32): [R, N].

    A: [R, K], the rows of the groups back to back, a scale per 128 elements of a row. B: [E, N, K], 128 x 128 blocks. M_array: uint32 [E],
    the rows of every group, on the device; None with one group (B may then be [N, K]): a plain matrix product. Rows past the last group are
    not written. K must be a multiple of 16. No gradients: grouped_linear_fp8 has them.
    """
    A, B = Fp8Blocks(*A), Fp8Blocks(*B)
    if B.values.dim() == 2 and B.scales.dim() == 2:
        B = Fp8Blocks(B.values[None], B.scales[None])
    assert A.values.dim() == 2 and B.values.dim() == 3, "A should be [R, K], B [E, N, K]"
    E, N, K = B.values.shape
    R = A.values.size(0)
    assert A.values.size(1) == K, "A and B should have the same reduction length"
    assert K % 16 == 0, "the reduction length should be a multiple of 16"
    assert block_rows_of(A) == 1 or R == 1, "A should have a scale per row and 128 elements"
    assert B.scales.shape == (E, ceil_divide(N, BLOCK_SIZE), scale_columns(K)) and block_rows_of(B), "B should have 128 x 128 blocks"
    assert output_dtype in _FLOATS, f"grouped_gemm_fp8 gives float32, float16 and bfloat16, not {output_dtype}"
    assert M_array is not None or E == 1, "several groups need M_array"
    _check_sizes(M_array, E)
    output = torch.empty(R, N, dtype=output_dtype, device=A.values.device)
    grouped_gemm_fp8_cuda(*A, *B, M_array, output)
    return output


class _GroupedLinearFp8(torch.autograd.Function):
    @staticmethod
    @ensure_contiguous
    def forward(ctx, x: torch.Tensor, weight: torch.Tensor, M_array: torch.Tensor, grad_enabled: bool) -> torch.Tensor:
        needs_x, needs_weight = (grad_enabled and n for n in ctx.needs_input_grad[:2])
        x8 = quantize_fp8(x)
        weight8, weight8_t = quantize_fp8(weight, BLOCK_SIZE, transposed=True) if needs_x else (quantize_fp8(weight, BLOCK_SIZE), None)
        output = grouped_gemm_fp8(x8, weight8, M_array, x.dtype)
        if needs_x or needs_weight:
            # x is kept in 8 bits, for the weight's gradient; the weight as its transposed copy, for x's
            ctx.save_for_backward(*(x8 if needs_weight else (None, None)), *(weight8_t or (None, None)), M_array)
        return output

    @staticmethod
    @ensure_contiguous
    def backward(ctx, output_grad: torch.Tensor) -> tuple[torch.Tensor | None, ...]:
        from ...modules.moe.cuda_implementation import grouped_gemm_ragged_cuda

        x_values, x_scales, weight_values, weight_scales, M_array = ctx.saved_tensors
        x_grad = weight_grad = None
        if ctx.needs_input_grad[0]:
            x_grad = grouped_gemm_fp8(quantize_fp8(output_grad), Fp8Blocks(weight_values, weight_scales), M_array, output_grad.dtype)
        if ctx.needs_input_grad[1]:
            x = dequantize_fp8(Fp8Blocks(x_values, x_scales), output_grad.dtype)
            E, N, K = M_array.numel(), output_grad.size(1), x.size(1)
            weight_grad = output_grad.new_empty(E, N, K)
            if x.size(0) == 0:
                weight_grad.zero_()
            else:
                grouped_gemm_ragged_cuda(output_grad, x, weight_grad, M_array, True, N, K, 0, True, False)
        return x_grad, weight_grad, None, None


def grouped_linear_fp8(x: torch.Tensor, weight: torch.Tensor, M_array: torch.Tensor) -> torch.Tensor:
    """y_e = x_e W_e^T for every group e with the product in 8 bits, from 16-bit tensors: x [R, K], rows of the groups back to back, weight
    [E, N, K], M_array uint32 [E] on the device, summing to R. x is quantised in blocks of 128 along its rows, the weight in 128 x 128 blocks.

    The gradient of x is the 8-bit product of output_grad, quantised along its rows, with the quantised weight; the gradient of the weight
    the 16-bit product of output_grad with the quantised x, which is all of x that is kept. K and N must be multiples of 16."""
    assert x.dim() == 2 and weight.dim() == 3 and x.size(1) == weight.size(2), "x should be [R, K], weight [E, N, K]"
    assert x.dtype == weight.dtype and x.dtype in (torch.float16, torch.bfloat16), "x and weight should both be float16 or bfloat16"
    assert weight.size(1) % 16 == 0 and weight.size(2) % 16 == 0, "both sides of the weight should be multiples of 16"
    assert weight.numel() > 0, "weight should not be empty"
    assert M_array is not None
    _check_sizes(M_array, weight.size(0))
    return _GroupedLinearFp8.apply(x, weight, M_array, torch.is_grad_enabled())
