"""Custom ops over fma_quantize_fp8, fma_dequantize_fp8 and fma_grouped_gemm_fp8 of libfma_hip.so."""

import torch

from ... import _lib
from ..._ops import hip_op


def _matrices(t: torch.Tensor) -> tuple[int, int, int]:
    """t [.., N, K] as (matrices, N, K)"""
    N, K = t.shape[-2:]
    E = 1
    for n in t.shape[:-2]:
        E *= n
    return E, N, K


def _check_blocks(values: torch.Tensor, scales: torch.Tensor, N: int, K: int, block_rows: int) -> None:
    assert values.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
    assert values.is_contiguous() and scales.is_contiguous()
    assert scales.shape == (*values.shape[:-2], -(-N // block_rows), 4 * -(-K // 512))


@hip_op("quantize_fp8_cuda", mutates_args={"values", "scales", "values_t", "scales_t"})
def quantize_fp8_cuda(
    x: torch.Tensor,
    values: torch.Tensor,
    scales: torch.Tensor,
    values_t: torch.Tensor | None,
    scales_t: torch.Tensor | None,
    block_rows: int,
) -> None:
    _lib.require_gpu(x, values, scales, values_t, scales_t)
    assert x.dim() >= 2 and x.is_contiguous() and values.shape == x.shape and block_rows in (1, 128)
    E, N, K = _matrices(x)
    _check_blocks(values, scales, N, K, block_rows)
    if values_t is not None:
        assert values_t.shape == (*x.shape[:-2], K, N)
        _check_blocks(values_t, scales_t, K, N, block_rows)
    if x.numel() == 0:
        return
    with _lib.on_device(x.device):
        rc = _lib.load().fma_quantize_fp8(
            x.data_ptr(), values.data_ptr(), scales.data_ptr(), _lib.ptr(values_t), _lib.ptr(scales_t), E, N, K, block_rows,
            _lib.dtype_code(x.dtype), _lib.current_stream(x.device),
        )  # fmt: skip
    _lib.check(rc, "quantize_fp8_cuda")


@hip_op("dequantize_fp8_cuda", mutates_args={"output"})
def dequantize_fp8_cuda(values: torch.Tensor, scales: torch.Tensor, output: torch.Tensor, block_rows: int) -> None:
    _lib.require_gpu(values, scales, output)
    assert values.dim() >= 2 and output.shape == values.shape and output.is_contiguous() and block_rows in (1, 128)
    E, N, K = _matrices(values)
    _check_blocks(values, scales, N, K, block_rows)
    if values.numel() == 0:
        return
    with _lib.on_device(values.device):
        rc = _lib.load().fma_dequantize_fp8(
            values.data_ptr(), scales.data_ptr(), output.data_ptr(), E, N, K, block_rows, _lib.dtype_code(output.dtype),
            _lib.current_stream(values.device),
        )  # fmt: skip
    _lib.check(rc, "dequantize_fp8_cuda")


@hip_op("grouped_gemm_fp8_cuda", mutates_args={"output"})
def grouped_gemm_fp8_cuda(
    A: torch.Tensor,
    A_scales: torch.Tensor,
    B: torch.Tensor,
    B_scales: torch.Tensor,
    M_array: torch.Tensor | None,
    output: torch.Tensor,
) -> None:
    _lib.require_gpu(A, A_scales, B, B_scales, M_array, output)
    E, N, K = B.shape
    R = A.size(0)
    assert A.shape == (R, K) and output.shape == (R, N) and output.is_contiguous()
    _check_blocks(A, A_scales, R, K, 1)
    _check_blocks(B, B_scales, N, K, 128)
    assert M_array is not None or E == 1
    assert M_array is None or (M_array.dtype == torch.uint32 and M_array.numel() == E and M_array.is_contiguous())
    for t in (A_scales, B, B_scales, M_array, output):
        assert t is None or t.device == A.device
    if output.numel() == 0:
        return
    with _lib.on_device(A.device):
        rc = _lib.load().fma_grouped_gemm_fp8(
            A.data_ptr(), A_scales.data_ptr(), B.data_ptr(), B_scales.data_ptr(), output.data_ptr(), _lib.ptr(M_array), E, R, N, K,
            _lib.dtype_code(output.dtype), _lib.current_stream(A.device),
        )  # fmt: skip
    _lib.check(rc, "grouped_gemm_fp8_cuda")
