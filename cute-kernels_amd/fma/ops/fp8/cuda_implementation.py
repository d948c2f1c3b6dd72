"""Custom ops over fma_quantize_fp8, fma_dequantize_fp8 and fma_grouped_gemm_fp8 of libfma_hip.so."""

import torch

from ... import _lib
from ..._ops import hip_op


def scales_dtype() -> torch.dtype:
    """float8_e8m0fnu; bytes in a traced function, whose compiler cannot write a tensor of that type by way of an operator"""
    return torch.uint8 if torch.compiler.is_compiling() else torch.float8_e8m0fnu


def operator_scales(scales: torch.Tensor) -> torch.Tensor:
    """scales as an operator takes them (see scales_dtype)"""
    return scales.view(torch.uint8) if torch.compiler.is_compiling() and scales.dtype is not torch.uint8 else scales


def is_scales_dtype(dtype: torch.dtype) -> bool:
    return dtype == torch.float8_e8m0fnu or dtype == torch.uint8


def _matrices(t: torch.Tensor) -> tuple[int, int, int]:
    """t [.., N, K] as (matrices, N, K)"""
    N, K = t.shape[-2:]
    E = 1
    for n in t.shape[:-2]:
        E *= n
    return E, N, K


def _check_blocks(values: torch.Tensor, scales: torch.Tensor, N: int, K: int, block_rows: int) -> None:
    assert values.dtype == torch.float8_e4m3fn and is_scales_dtype(scales.dtype)
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


@hip_op("grouped_linear_fp8_cuda", mutates_args={"x_values", "x_scales", "weight_values", "weight_scales", "weight_t_values", "weight_t_scales", "output"})
def grouped_linear_fp8_cuda(
    x: torch.Tensor, weight: torch.Tensor, M_array: torch.Tensor, x_values: torch.Tensor, x_scales: torch.Tensor,
    weight_values: torch.Tensor, weight_scales: torch.Tensor, weight_t_values: torch.Tensor | None, weight_t_scales: torch.Tensor | None,
    output: torch.Tensor,
) -> None:  # fmt: skip
    """quantize_fp8 of x and of weight (with its transposed copy if that is asked for) and grouped_gemm_fp8 of the two, as one call"""
    _lib.require_gpu(x, weight, M_array, x_values, x_scales, weight_values, weight_scales, weight_t_values, weight_t_scales, output)
    E, N, K = weight.shape
    R = x.size(0)
    assert x.shape == (R, K) == x_values.shape and weight_values.shape == weight.shape and output.shape == (R, N)
    assert x.dtype == weight.dtype == output.dtype and x.is_contiguous() and weight.is_contiguous() and output.is_contiguous()
    assert M_array.dtype == torch.uint32 and M_array.numel() == E and M_array.is_contiguous()
    _check_blocks(x_values, x_scales, R, K, 1)
    _check_blocks(weight_values, weight_scales, N, K, 128)
    if weight_t_values is not None:
        assert weight_t_values.shape == (E, K, N)
        _check_blocks(weight_t_values, weight_t_scales, K, N, 128)
    for t in (weight, M_array, x_values, x_scales, weight_values, weight_scales, output):
        assert t.device == x.device
    with _lib.on_device(x.device):
        rc = _lib.load().fma_grouped_linear_fp8(
            x.data_ptr(), weight.data_ptr(), x_values.data_ptr(), x_scales.data_ptr(), weight_values.data_ptr(), weight_scales.data_ptr(),
            _lib.ptr(weight_t_values), _lib.ptr(weight_t_scales), output.data_ptr(), M_array.data_ptr(), E, R, N, K,
            _lib.dtype_code(x.dtype), _lib.current_stream(x.device),
        )  # fmt: skip
    _lib.check(rc, "grouped_linear_fp8_cuda")


@hip_op("grouped_linear_fp8_backward_cuda", mutates_args={"x_grad", "weight_grad"})
def grouped_linear_fp8_backward_cuda(
    output_grad: torch.Tensor, x_values: torch.Tensor | None, x_scales: torch.Tensor | None, weight_t_values: torch.Tensor | None,
    weight_t_scales: torch.Tensor | None, M_array: torch.Tensor, K: int, x_grad: torch.Tensor | None, weight_grad: torch.Tensor | None,
) -> None:  # fmt: skip
    _lib.require_gpu(output_grad, x_values, x_scales, weight_t_values, weight_t_scales, M_array, x_grad, weight_grad)
    R, N = output_grad.shape
    E = M_array.numel()
    assert output_grad.is_contiguous() and M_array.dtype == torch.uint32 and M_array.is_contiguous()
    if x_grad is not None:
        assert x_grad.shape == (R, K) and x_grad.dtype == output_grad.dtype and x_grad.is_contiguous()
        assert weight_t_values.shape == (E, K, N)
        _check_blocks(weight_t_values, weight_t_scales, K, N, 128)
    if weight_grad is not None:
        assert weight_grad.shape == (E, N, K) and weight_grad.dtype == output_grad.dtype and weight_grad.is_contiguous()
        assert x_values.shape == (R, K)
        _check_blocks(x_values, x_scales, R, K, 1)
    lib = _lib.load()
    with _lib.on_device(output_grad.device):
        nbytes = lib.fma_grouped_linear_fp8_bwd_workspace_bytes(R, N, K)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=output_grad.device)
        rc = lib.fma_grouped_linear_fp8_bwd(
            output_grad.data_ptr(), _lib.ptr(x_values), _lib.ptr(x_scales), _lib.ptr(weight_t_values), _lib.ptr(weight_t_scales),
            _lib.ptr(x_grad), _lib.ptr(weight_grad), M_array.data_ptr(), E, R, N, K, workspace.data_ptr(), nbytes,
            _lib.dtype_code(output_grad.dtype), _lib.current_stream(output_grad.device),
        )  # fmt: skip
    _lib.check(rc, "grouped_linear_fp8_backward_cuda")
