"""The 8-bit operators without a GPU: the oracle against torch's own e4m3, refusals of the C entry points and of the public functions."""

import ctypes

import pytest
import torch

import fma
from fma import Fp8Blocks, MoE, grouped_gemm_fp8, grouped_linear_fp8, quantize_expert_weights, quantize_fp8, swiglu_experts_fp8, swiglu_packed
from fma.modules.moe.fp8_implementation import buffer_bytes
from oracle import fp8_oracle as O


def test_oracle_rounds_as_torch_does():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4000, generator=g) * torch.exp2(torch.randint(-12, 9, (4000,), generator=g).float())
    x = x.clamp(-448, 448)
    assert torch.equal(O.round_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    borders = torch.tensor([0.0, 2.0**-10, 3 * 2.0**-10, 2.0**-9, 17.0, 18.0, 19.0, 440.0, 448.0])  # ties among them
    assert torch.equal(O.round_e4m3(borders.double()), borders.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("amax,byte", [(448.0, 127), (448.001, 128), (224.0, 126), (0.0, 1), (1.0, 119), (1.75, 119), (1.7501, 120), (2.0**-149, 1)])
def test_oracle_scales(amax, byte):
    values, scales = O.quantize(torch.tensor([[0.0, -amax]], dtype=torch.float64).float())
    assert int(scales[0, 0]) == byte and scales[0, 1:].eq(127).all()
    assert float(values.abs().max()) <= 448


def _pointer():
    buf = ctypes.create_string_buffer(4096 + 16)
    return buf, (ctypes.addressof(buf) + 15) & ~15  # a 16-byte aligned, non-NULL (host) address: never dereferenced


def _err(lib) -> str:
    return lib.fma_last_error_string().decode()


def test_quantize_and_swiglu_validation(lib):
    buf, p = _pointer()
    assert [lib.fma_fp8_scale_pitch(k) for k in (0, 1, 128, 512, 513, 2880)] == [0, 4, 4, 4, 8, 24]
    assert lib.fma_quantize_fp8(p, p, p, None, None, 1, 4, 128, 1, 7, None) == -2
    assert lib.fma_quantize_fp8(p, p, p, None, None, 1, 4, 128, 64, 2, None) == -3 and "1 or 128" in _err(lib)
    assert lib.fma_quantize_fp8(p, p, p, p, p, 1, 4, 128, 1, 2, None) == -8  # a transposed copy of rows
    assert lib.fma_quantize_fp8(p, p, p, p, None, 1, 4, 128, 128, 2, None) == -1
    assert lib.fma_quantize_fp8(p, p, None, None, None, 1, 4, 128, 1, 2, None) == -1
    assert lib.fma_quantize_fp8(p, p, p, None, None, 1, 4, 0, 1, 2, None) == -3
    assert lib.fma_quantize_fp8(p, p, p, None, None, 1, 1 << 40, 1 << 20, 1, 2, None) == -5
    assert lib.fma_quantize_fp8(p + 1, p, p, None, None, 1, 4, 128, 1, 2, None) == -6
    assert lib.fma_quantize_fp8(None, None, None, None, None, 1, 0, 128, 1, 2, None) == 0
    assert lib.fma_dequantize_fp8(p, p, None, 1, 4, 128, 1, 2, None) == -1
    assert lib.fma_dequantize_fp8(p, p, p, 1, 4, 128, 3, 2, None) == -3
    assert lib.fma_dequantize_fp8(None, None, None, 0, 4, 128, 128, 2, None) == 0
    assert lib.fma_swiglu_fp8_forward(p, p, p, p, 4, 0, 2, None) == -3
    assert lib.fma_swiglu_fp8_forward(p, p, p, None, 4, 8, 2, None) == -1
    assert lib.fma_swiglu_fp8_backward(p, p, p, p, 4, 8, 5, None) == -2
    assert lib.fma_swiglu_fp8_backward(None, None, None, None, 0, 8, 2, None) == 0


def test_product_validation(lib):
    buf, p = _pointer()
    product = lib.fma_grouped_gemm_fp8
    assert product(p, p, p, p, p, p, 4, 10, 64, 120, 2, None) == -3 and "multiple of 16" in _err(lib)
    assert product(p, p, p, p, p, p, 1025, 10, 64, 128, 2, None) == -4
    assert product(p, p, p, p, p, p, 4, 10, 64, 1 << 21, 2, None) == -5
    assert product(p, p, p, p, p, p, 4, 1 << 31, 64, 128, 2, None) == -5
    assert product(p, p, p, p, p, p, 1, 10, 1 << 20, 1 << 12, 2, None) == -5  # a matrix of 2^32 bytes
    assert product(p, p, p, p, p, p, 4, 10, 64, 128, 9, None) == -2
    assert product(p, p, p, p, p, None, 4, 10, 64, 128, 2, None) == -1  # several groups without their sizes
    assert product(p, None, p, p, p, p, 4, 10, 64, 128, 2, None) == -1
    assert product(p + 4, p, p, p, p, p, 4, 10, 64, 128, 2, None) == -6
    assert product(p, p + 1, p, p, p, p, 4, 10, 64, 128, 2, None) == -6 and "4 bytes" in _err(lib)
    for empty in ((0, 10, 64), (4, 0, 64), (4, 10, 0)):
        assert product(None, None, None, None, None, p, *empty, 128, 2, None) == 0


def test_linear_validation(lib):
    buf, p = _pointer()

    def backward(R=8, N=64, K=32, dtype=2, dy=p, x=p, wt=p, size=1 << 30):
        return lib.fma_grouped_linear_fp8_bwd(dy, x, x, wt, wt, p, p, p, 2, R, N, K, p, size, dtype, None)

    assert lib.fma_grouped_linear_fp8(p, p, p, p, p, p, None, None, p, p, 2, 8, 64, 32, 0, None) == -2
    assert lib.fma_grouped_linear_fp8(p, p, p, p, p, p, None, None, p, p, 2, 8, 64, 24, 2, None) == -3
    assert lib.fma_grouped_linear_fp8(p, p, p, p, p, p, p, None, p, p, 2, 8, 64, 32, 2, None) == -1
    assert backward(dtype=0) == -2 and backward(N=40) == -3 and backward(dy=None) == -1 and backward(x=None) == -1 and backward(wt=None) == -1
    assert backward(size=64) == -7 and backward(R=0) == 0
    assert lib.fma_grouped_linear_fp8_bwd_workspace_bytes(8, 64, 32) == 512 + 256 + 512


def test_experts_validation(lib):
    buf, p = _pointer()

    def forward(T=4, k=2, E=4, H=64, I=32, dtype=2, id_bytes=4, ids=p, buffer=p, buffer_size=1 << 30, workspace_size=1 << 30):
        return lib.fma_swiglu_experts_fp8(p, p, ids, id_bytes, p, p, p, p, p, T, k, E, H, I, 0, buffer, buffer_size, p, workspace_size, dtype, None)

    def backward(T=4, k=2, E=4, H=64, I=32, dtype=2, id_bytes=4, buffer_size=1 << 30, workspace_size=1 << 30):
        return lib.fma_swiglu_experts_fp8_bwd(p, p, p, id_bytes, p, p, p, p, p, buffer_size, p, p, p, p, T, k, E, H, I, p, workspace_size, dtype, None)

    for call in (forward, backward):
        assert call(dtype=0) == -2 and "16-bit" in _err(lib)
        assert call(H=72) == -3 and call(I=40) == -3 and "multiples of 16" in _err(lib)
        assert call(E=1025) == -4 and call(k=0) == -3 and call(id_bytes=2) == -2
        assert call(T=1 << 30, H=16) == -5 and call(T=1 << 20, k=1 << 12) == -5
        assert call(buffer_size=64) == -7 and "buffer" in _err(lib)
        assert call(workspace_size=4) == -7 and "workspace" in _err(lib)
        assert call(T=0) == 0
    assert forward(ids=None) == -1 and forward(buffer=None) == -1 and forward(ids=p + 2) == -6
    for sizes in ((1, 1, 1, 16, 16), (37, 2, 6, 256, 208), (8192, 8, 64, 2048, 1408), (3, 3, 5, 528, 1040)):
        assert lib.fma_swiglu_experts_fp8_buffer_bytes(*sizes, 1) == buffer_bytes(*sizes)
    assert lib.fma_swiglu_experts_fp8_buffer_bytes(8192, 8, 64, 2048, 1408, 0) < buffer_bytes(8192, 8, 64, 2048, 1408)


def _blocks(*shape, rows=1, K=None):
    *batch, N, K = shape
    return Fp8Blocks(
        torch.empty(shape, dtype=torch.float8_e4m3fn), torch.empty(*batch, -(-N // rows), 4 * -(-K // 512), dtype=torch.float8_e8m0fnu)
    )


def _sizes(*m):
    return torch.tensor(m, dtype=torch.int32).view(torch.uint32)


def test_refusals_of_the_public_functions():
    x = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        quantize_fp8(x)
    for bad in (lambda: quantize_fp8(x, 64), lambda: quantize_fp8(x.long()), lambda: quantize_fp8(x, 1, transposed=True),
                lambda: quantize_fp8(x[0], 128), lambda: quantize_fp8(x[:, :0]), lambda: quantize_fp8(x.double())):  # fmt: skip
        with pytest.raises(AssertionError):
            bad()
    a, b, sizes = _blocks(8, 64), _blocks(2, 48, 64, rows=128), _sizes(4, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        grouped_gemm_fp8(a, b, sizes)
    for bad in (lambda: grouped_gemm_fp8(a, b), lambda: grouped_gemm_fp8(a, b, _sizes(8)), lambda: grouped_gemm_fp8(a, b, sizes.view(torch.int32)),
                lambda: grouped_gemm_fp8(_blocks(8, 80), b, sizes), lambda: grouped_gemm_fp8(a, _blocks(2, 48, 64), sizes),
                lambda: grouped_gemm_fp8(_blocks(300, 64, rows=128), b, sizes), lambda: grouped_gemm_fp8(a, b, sizes, torch.float64),
                lambda: grouped_gemm_fp8(_blocks(8, 72), _blocks(2, 48, 72, rows=128), sizes),
                lambda: grouped_gemm_fp8(Fp8Blocks(a.values.float(), a.scales), b, sizes),
                lambda: grouped_gemm_fp8(Fp8Blocks(a.values, a.scales.view(torch.uint8)), b, sizes),
                lambda: fma.dequantize_fp8(a, torch.float64), lambda: fma.dequantize_fp8(Fp8Blocks(a.values, a.scales[:, :2]))):  # fmt: skip
        with pytest.raises(AssertionError):
            bad()
    x, w = torch.zeros(8, 64).bfloat16(), torch.zeros(2, 48, 64).bfloat16()
    for bad in (lambda: grouped_linear_fp8(x, w.half(), sizes), lambda: grouped_linear_fp8(x.float(), w.float(), sizes),
                lambda: grouped_linear_fp8(x, w[:, :40], sizes), lambda: grouped_linear_fp8(x, w, None), lambda: grouped_linear_fp8(x[:, :32], w, sizes)):  # fmt: skip
        with pytest.raises(AssertionError):
            bad()
    for bad in (torch.zeros(4, 7), torch.zeros(4, 0), torch.zeros(4, 8).double()):
        with pytest.raises(AssertionError):
            fma.swiglu_packed_fp8(bad)
    with pytest.raises(ValueError, match="kernel_backend"):
        fma.swiglu_packed_fp8(torch.zeros(4, 8), kernel_backend_forward=fma.KernelBackend.torch)


def test_refusals_of_the_expert_path():
    T, H, I, E, k = 4, 64, 32, 3, 2
    x, gates, ids = torch.zeros(T, H).bfloat16(), torch.zeros(T, k).bfloat16(), torch.zeros(T, k, dtype=torch.int32)
    w1, w2 = torch.zeros(E, 2 * I, H).bfloat16(), torch.zeros(E, H, I).bfloat16()
    q1, q2 = _blocks(E, 2, I, H, rows=128), _blocks(E, H, I, rows=128)
    for operands in ((w1, w2), (q1, q2)):
        with pytest.raises(RuntimeError, match="GPU only"):
            swiglu_experts_fp8(x, gates, ids, *operands)
    with pytest.raises(RuntimeError, match="no gradients"):
        swiglu_experts_fp8(x.clone().requires_grad_(), gates, ids, q1, q2)
    bad = [
        (x.float(), gates, ids, w1, w2), (x, gates.float(), ids, w1, w2), (x, gates, ids.short(), w1, w2), (x, gates[:, :1], ids, w1, w2),
        (x[:3], gates, ids, w1, w2), (x, gates, ids, w1, q2), (x, gates, ids, q1, w2), (x, gates, ids, w1.half(), w2),
        (x, gates, ids, w1[:, :-1], w2), (x, gates, ids, w1, w2[:2]), (x, gates, ids, _blocks(E, 2 * I, H, rows=128), q2),
        (x[:, :56], gates, ids, w1[:, :, :56], w2[:, :56]), (x, gates[:, :0], ids[:, :0], w1, w2), (x, gates, ids, q1, _blocks(E, H, I)),
    ]  # fmt: skip
    for args in bad:
        with pytest.raises((AssertionError, RuntimeError)) as info:
            swiglu_experts_fp8(*args)
        assert info.type is AssertionError or "GPU only" in str(info.value)
    moe = MoE(E, k, H, I, swiglu_packed, True, False, 0.02)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        moe.quantize_experts()
    assert not moe.fp8_experts and "fp8" not in str(list(moe.state_dict()))
    with pytest.raises(RuntimeError, match="GPU only"):
        quantize_expert_weights(w1, w2)


def test_refusals_of_serving_with_tangents_and_without_experts():
    x, gates, ids = torch.zeros(3, 32).bfloat16(), torch.zeros(3, 2).bfloat16(), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(AssertionError, match="an expert"):
        fma.swiglu_experts_fp8(x, gates, ids, torch.zeros(0, 64, 32).bfloat16(), torch.zeros(0, 32, 32).bfloat16())

    def blocks(*shape):
        scales = torch.full((*shape[:-2], 1, 4), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        return fma.Fp8Blocks(torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn), scales)

    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no gradients"):
            fma.swiglu_experts_fp8(dual, gates, ids, blocks(2, 2, 32, 32), blocks(2, 32, 32))


def test_refusal_of_parameters_made_in_inference_mode():
    with torch.inference_mode():
        moe = fma.MoE(4, 2, 32, 32, fma.swiglu_packed, True, False, 0.02).to(torch.bfloat16)
    with pytest.raises(ValueError, match="inference mode"):
        moe.quantize_experts()


def test_launches_that_would_not_fit_are_refused_up_front(lib):
    """a launch has fewer than 2^32 threads: sizes that need more are refused before anything is enqueued"""
    buf, p = _pointer()
    assert lib.fma_quantize_fp8(p, p, p, None, None, 1 << 24, 1, 128, 128, 2, None) == -5 and "2^24" in _err(lib)
    assert lib.fma_quantize_fp8(p, p, p, p, p, 1 << 12, 1 << 12, 1 << 14, 128, 2, None) == -5

    def forward(T, k, H=16, I=16):
        return lib.fma_swiglu_experts_fp8(p, p, p, 4, p, p, p, p, p, T, k, 4, H, I, 0, p, 0, p, 0, 2, None)

    def backward(T, k, H=16, I=16):
        return lib.fma_swiglu_experts_fp8_bwd(p, p, p, 4, p, p, p, p, p, 0, p, p, p, p, T, k, 4, H, I, p, 0, 2, None)

    for call in (forward, backward):
        assert call(1 << 24, 1) == -5 and "T < 2^24" in _err(lib)
        assert call(1 << 22, 16) == -5 and call((1 << 22) - 1, 16) == -7  # (the next refusal: no buffer)
        assert call((1 << 24) - 1, 1) == -7 and call(1 << 22, 8, I=1 << 13) == -5 and call(1 << 22, 8, I=1 << 10) == -7


def test_a_layer_saved_before_it_had_8_bit_experts_still_loads_and_runs():
    """a pickled module comes back with the attributes that it was saved with"""
    moe = MoE(4, 2, 32, 32, swiglu_packed, True, False, 0.02).to(torch.bfloat16)
    for name in ("fp8_experts", "_fp8_weights"):
        moe.__dict__.pop(name, None)
    loaded = MoE.__new__(MoE)
    loaded.__setstate__(moe.__dict__.copy())
    assert loaded.fp8_experts is False
    with pytest.raises(RuntimeError, match="GPU only"):
        loaded(torch.zeros(3, 32).bfloat16(), kernel_backend=fma.KernelBackend.cuda)
    with pytest.raises(RuntimeError, match="GPU only"):
        loaded.quantize_experts()
