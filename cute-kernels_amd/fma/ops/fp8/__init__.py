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
from .cuda_implementation import (
    dequantize_fp8_cuda,
    grouped_gemm_fp8_cuda,
    grouped_linear_fp8_backward_cuda,
    grouped_linear_fp8_cuda,
    operator_scales,
    quantize_fp8_cuda,
    scales_dtype,
)

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
        torch.empty(*batch, ceil_divide(N, block_rows), scale_columns(K), dtype=scales_dtype(), device=device),
    )


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
    one_row = x.dim() == 1
    shape = (1, x.size(0)) if one_row else tuple(x.shape)
    assert not transposed or shape[-2] > 0, "columns must not be empty"
    x = x.detach().contiguous().view(shape)
    blocks = _empty_blocks(shape, block_rows, x.device)
    other = _empty_blocks((*shape[:-2], shape[-1], shape[-2]), block_rows, x.device) if transposed else None
    quantize_fp8_cuda(x, *blocks, *(other or (None, None)), block_rows)
    if torch.compiler.is_compiling():
        blocks, other = (b and Fp8Blocks(b.values, b.scales.view(torch.float8_e8m0fnu)) for b in (blocks, other))
    if one_row:
        return Fp8Blocks(blocks.values[0], blocks.scales[0])
    return blocks if other is None else (blocks, other)


def block_rows_of(blocks: Fp8Blocks) -> int:
    """1 or 128, from the shapes; raises if they do not fit each other"""
    values, scales = blocks
    assert values.dtype is torch.float8_e4m3fn and scales.dtype is torch.float8_e8m0fnu, "values in e4m3, scales in e8m0"
    assert values.dim() >= 2, "values should have two dimensions at least"
    *batch, N, K = values.shape
    for block_rows in (1, BLOCK_SIZE):
        if K > 0 and scales.shape == (*batch, ceil_divide(N, block_rows), scale_columns(K)):
            return block_rows
    raise AssertionError(f"scales of shape {tuple(scales.shape)} do not fit values of shape {tuple(values.shape)}")


def dequantize_fp8(blocks: Fp8Blocks, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that the blocks stand for, rounded to dtype: exact in float32 and bfloat16. What a dtype's largest numbers round up to in
    8 bits, 65536 and 2^128 (numbers of 63488 and of 248 * 2^120 and more), becomes its largest number."""
    assert dtype in _FLOATS, f"dequantize_fp8 gives float32, float16 and bfloat16, not {dtype}"
    values, scales = (t.contiguous() for t in blocks)
    one_row = values.dim() == 1
    if one_row:
        values, scales = values[None], scales[None]
    block_rows = block_rows_of((values, scales))
    output = torch.empty(values.shape, dtype=dtype, device=values.device)
    dequantize_fp8_cuda(values, operator_scales(scales), output, block_rows)
    return output[0] if one_row else output


def _check_sizes(M_array: torch.Tensor | None, E: int) -> None:
    if M_array is not None:
        assert M_array.dtype == torch.uint32 and M_array.shape == (E,), "M_array should be uint32 with one entry per group"


def grouped_gemm_fp8(
    A: Fp8Blocks, B: Fp8Blocks, M_array: torch.Tensor | None = None, output_dtype: torch.dtype = torch.bfloat16
) -> torch.Tensor:
    """D_e = A_e B_e^T for every group e, fp32 sums, rounded once to output_dtype (bfloat16, float16 or float32): [R, N].

    A: [R, K], the rows of the groups back to back, a scale per 128 elements of a row. B: [E, N, K], 128 x 128 blocks. M_array: uint32 [E],
    the rows of every group, on the device; None with one group (B may then be [N, K]): a plain matrix product. Rows past the last group are
    not written. K must be a multiple of 16. No gradients: grouped_linear_fp8 has them.
    """
    (a, a_scales), (b, b_scales) = A, B
    if b.dim() == 2 and b_scales.dim() == 2:
        b, b_scales = b[None], b_scales[None]
    assert a.dim() == 2 and b.dim() == 3, "A should be [R, K], B [E, N, K]"
    (R, K), (E, N, _) = a.shape, b.shape
    assert b.size(2) == K, "A and B should have the same reduction length"
    assert K > 0 and K % 16 == 0, "the reduction length should be a multiple of 16"
    assert a.dtype is b.dtype is torch.float8_e4m3fn and a_scales.dtype is b_scales.dtype is torch.float8_e8m0fnu, (
        "values in e4m3, scales in e8m0"
    )
    columns = scale_columns(K)
    assert a_scales.shape == (R, columns), "A should have a scale per row and 128 elements"
    assert b_scales.shape == (E, ceil_divide(N, BLOCK_SIZE), columns), "B should have 128 x 128 blocks"
    assert output_dtype in _FLOATS, f"grouped_gemm_fp8 gives float32, float16 and bfloat16, not {output_dtype}"
    if M_array is not None:
        _check_sizes(M_array, E)
        M_array = M_array.contiguous()
    else:
        assert E == 1, "several groups need M_array"
    output = torch.empty(R, N, dtype=output_dtype, device=a.device)
    a_scales, b_scales = operator_scales(a_scales.contiguous()), operator_scales(b_scales.contiguous())
    grouped_gemm_fp8_cuda(a.contiguous(), a_scales, b.contiguous(), b_scales, M_array, output)
    return output


class _GroupedLinearFp8(torch.autograd.Function):
    @staticmethod
    @ensure_contiguous
    def forward(ctx, x: torch.Tensor, weight: torch.Tensor, M_array: torch.Tensor, grad_enabled: bool) -> torch.Tensor:
        needs_x, needs_weight = (grad_enabled and n for n in ctx.needs_input_grad[:2])
        E, N, K = weight.shape
        x8 = _empty_blocks(x.shape, 1, x.device)
        weight8 = _empty_blocks(weight.shape, BLOCK_SIZE, x.device)
        weight8_t = _empty_blocks((E, K, N), BLOCK_SIZE, x.device) if needs_x else (None, None)
        output = x.new_empty(x.size(0), N)
        grouped_linear_fp8_cuda(x, weight, M_array, *x8, *weight8, *weight8_t, output)
        if needs_x or needs_weight:
            # x is kept in 8 bits, for the weight's gradient; the weight as its transposed copy, for x's
            ctx.save_for_backward(*(x8 if needs_weight else (None, None)), *weight8_t, M_array)
            ctx.K = K
        return output

    @staticmethod
    @ensure_contiguous
    def backward(ctx, output_grad: torch.Tensor) -> tuple[torch.Tensor | None, ...]:
        *saved, M_array = ctx.saved_tensors
        (R, N), K = output_grad.shape, ctx.K
        x_grad = output_grad.new_empty(R, K) if ctx.needs_input_grad[0] else None
        weight_grad = None
        if ctx.needs_input_grad[1]:
            weight_grad = (output_grad.new_empty if R else output_grad.new_zeros)(M_array.numel(), N, K)
        if R:
            grouped_linear_fp8_backward_cuda(output_grad, *saved, M_array, K, x_grad, weight_grad)
        return x_grad, weight_grad, None, None


def grouped_linear_fp8(x: torch.Tensor, weight: torch.Tensor, M_array: torch.Tensor) -> torch.Tensor:
    """y_e = x_e W_e^T for every group e with the product in 8 bits, from 16-bit tensors: x [R, K], rows of the groups back to back, weight
    [E, N, K], M_array uint32 [E] on the device, summing to R (rows past the last group are not written, of the gradient neither; sizes past R
    are cut to it). x is quantised in blocks of 128 along its rows, the weight in 128 x 128 blocks.

    The gradient of x is the 8-bit product of output_grad, quantised along its rows, with the quantised weight; the gradient of the weight
    the 16-bit product of output_grad with the quantised x, which is all of x that is kept. K and N must be multiples of 16."""
    assert x.dim() == 2 and weight.dim() == 3 and x.size(1) == weight.size(2), "x should be [R, K], weight [E, N, K]"
    assert x.dtype == weight.dtype and x.dtype in (torch.float16, torch.bfloat16), "x and weight should both be float16 or bfloat16"
    assert weight.size(1) % 16 == 0 and weight.size(2) % 16 == 0, "both sides of the weight should be multiples of 16"
    assert weight.numel() > 0, "weight should not be empty"
    assert M_array is not None
    _check_sizes(M_array, weight.size(0))
    return _GroupedLinearFp8.apply(x, weight, M_array, torch.is_grad_enabled())
