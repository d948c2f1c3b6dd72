"""The 8-bit block format and its products on the GPU against the 64-bit oracle: conversion bit by bit, products to the rounding of their sums."""

import pytest
import torch

import fma
from fma import Fp8Blocks, dequantize_fp8, grouped_gemm_fp8, grouped_linear_fp8, quantize_fp8
from gpu_util import DEV
from oracle import fp8_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _bytes(t: torch.Tensor) -> torch.Tensor:
    return t.cpu().contiguous().view(torch.uint8)


def _values(t: torch.Tensor) -> torch.Tensor:
    return t.cpu().double()


def _hard(g, *shape) -> torch.Tensor:
    """magnitudes over many powers of two, zeros among them, some blocks at the format's borders"""
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-18, 6, shape, generator=g).float())
    x[torch.rand(*shape, generator=g) < 0.1] = 0.0
    return x


def _sizes(counts) -> torch.Tensor:
    return torch.tensor(counts, dtype=torch.int32, device=DEV).view(torch.uint32)


# ---- conversion -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (1, 16), (3, 127), (2, 128), (5, 144), (9, 500), (4, 512), (3, 528), (2, 1040), (33, 2880)])
def test_quantize_rows(dtype, N, K):
    x = _hard(torch.Generator().manual_seed(N * K), N, K).to(dtype)
    values, scales = quantize_fp8(x.to(DEV))
    expect, expect_scales = O.quantize(x)
    assert values.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
    assert torch.equal(_bytes(scales), expect_scales)
    assert torch.equal(_values(values), expect)
    back = dequantize_fp8(Fp8Blocks(values, scales), torch.float32)
    assert torch.equal(_values(back), O.dequantize(expect, expect_scales).float().double())
    if dtype is not torch.float32:
        back16 = dequantize_fp8(Fp8Blocks(values, scales), dtype)
        assert torch.equal(back16.cpu(), back.cpu().to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,N,K", [(1, 1, 1), (1, 128, 128), (2, 130, 144), (3, 24, 8), (1, 257, 513), (2, 256, 640), (1, 8, 1040)])
def test_quantize_blocks_and_their_transposed_copy(dtype, E, N, K):
    x = _hard(torch.Generator().manual_seed(N + K), E, N, K).to(dtype)
    (values, scales), (values_t, scales_t) = quantize_fp8(x.to(DEV), 128, transposed=True)
    alone = quantize_fp8(x.to(DEV), 128)
    assert torch.equal(_bytes(alone.values), _bytes(values)) and torch.equal(_bytes(alone.scales), _bytes(scales))
    for e in range(E):
        expect, expect_scales = O.quantize(x[e], 128)
        assert torch.equal(_values(values[e]), expect) and torch.equal(_bytes(scales[e]), expect_scales)
        t, t_scales = O.quantize(x[e].t(), 128)
        assert torch.equal(_values(values_t[e]), t) and torch.equal(_bytes(scales_t[e]), t_scales)
        back = dequantize_fp8(Fp8Blocks(values, scales), torch.float32)[e]
        assert torch.equal(_values(back), O.dequantize(expect, expect_scales, 128).float().double())


def test_quantize_extremes():
    """the borders of a scale, zeros, the smallest and largest numbers, infinities and NaN: the block, and only it, is NaN"""
    big, tiny = torch.finfo(torch.float32).max, 2.0**-149
    cases = [448.0, 448.0 + 2.0**-15, 447.999, 224.0, 224.00002, 0.0, tiny, 2.0**-126, 448.0 * 2.0**-126, 2.0**-117 * 1.76, big, 1.0]
    x = torch.zeros(len(cases) + 3, 256)
    for i, c in enumerate(cases):
        x[i, 5] = -c
        x[i, 6] = c / 3
        x[i, 200] = 1.0
    x[-3, 7], x[-2, 7], x[-1, 130] = float("inf"), float("nan"), -float("inf")
    for rows in (1, 128):
        blocks = quantize_fp8(x.to(DEV), rows)
        expect, scales = O.quantize(x, rows)
        assert torch.equal(_bytes(blocks.scales), scales)
        assert torch.equal(torch.nan_to_num(_values(blocks.values), nan=1e9), torch.nan_to_num(expect, nan=1e9))
    back = dequantize_fp8(quantize_fp8(x.to(DEV)), torch.float32).cpu()
    assert back[-3, :128].isnan().all() and back[-2, :128].isnan().all() and back[-1, 128:].isnan().all()
    assert not back[-3:, 128:][:2].isnan().any() and not back[-1, :128].isnan().any() and not back[:-3].isnan().any()


def test_quantize_shapes_and_strides():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 5, 320, generator=g).bfloat16().to(DEV)
    a = quantize_fp8(x)
    assert a.values.shape == x.shape and a.scales.shape == (6, 5, 4)
    b = quantize_fp8(x.transpose(0, 1))
    assert torch.equal(_bytes(b.values), _bytes(a.values.view(torch.uint8).transpose(0, 1)))
    c = quantize_fp8(x[2, 3])
    assert c.values.shape == (320,) and torch.equal(_bytes(c.values), _bytes(a.values[2, 3]))
    assert torch.equal(dequantize_fp8(c), dequantize_fp8(a)[2, 3])
    flat = torch.randn(700, generator=g).bfloat16().to(DEV)
    unaligned = quantize_fp8(flat[1:641])  # two bytes past a 16-byte border
    assert torch.equal(_bytes(unaligned.values), _bytes(quantize_fp8(flat[1:641].clone()).values))
    for shape in ((0, 320), (4, 0, 320)):
        empty = quantize_fp8(torch.empty(shape, device=DEV))
        assert empty.values.shape == shape and dequantize_fp8(empty).shape == shape


# ---- products -------------------------------------------------------------------------------------------------------


def _operands(counts, N, K, seed=0, rows=None):
    g = torch.Generator().manual_seed(seed)
    R = sum(counts) if rows is None else rows
    x = torch.randn(R, K, generator=g) * torch.exp(0.7 * torch.randn(K, generator=g))
    w = 0.05 * torch.randn(len(counts), N, K, generator=g) * torch.exp(0.7 * torch.randn(len(counts), 1, K, generator=g))
    return x, w


def _largest_of_eight(t):
    return torch.nn.functional.pad(t.abs(), (0, -t.size(1) % 8)).unflatten(1, (-1, 8)).amax(2)


def _check_product(got, x, w, counts, dtype):
    """x, w: the numbers that the operands stand for.

    The matrix instruction for 8-bit operands (the scaled and the plain one alike, measured with single products) brings each eight
    neighbouring products to the exponent of the largest, 2^E <= |a b|, and cuts what lies below 2^(E - 13) off every one of them: the
    largest has six bits after its point and loses nothing, the seven others less than 2^(E - 13) each, in all under
    7 * 2^-13 * max |a| * max |b| for every eight. Their sums are fp32 sums of at most K terms in any order, one ulp lost per addition
    at most; then half a step of the output's type."""
    first = 0
    for e, m in enumerate(counts):
        rows = slice(first, first + m)
        exact, size = x[rows] @ w[e].t(), x[rows].abs() @ w[e].abs().t()
        sums = x.size(1) * 2.0**-23 * size + 7 * 2.0**-13 * (_largest_of_eight(x[rows]) @ _largest_of_eight(w[e]).t())
        bound = sums + torch.finfo(dtype).eps / 2 * (exact.abs() + sums)
        bound += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a step of a subnormal result
        assert bool(((got[rows].cpu().double() - exact).abs() <= bound).all()), (e, m)
        first += m


SHAPES = [
    ([1], 16, 16), ([1], 1, 128), ([3], 7, 144), ([17], 130, 128), ([256], 256, 256), ([257], 264, 384), ([300, 0, 5], 520, 400),
    ([0, 0, 1], 40, 2064), ([64, 255, 256, 257, 1], 256, 640), ([2, 1, 0, 9, 30, 3], 96, 512), ([700], 300, 1024), ([513, 40], 128, 2880),
]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,N,K", SHAPES)
def test_grouped_gemm(dtype, counts, N, K):
    x, w = _operands(counts, N, K, seed=N + K)
    a, b = quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128)
    got = grouped_gemm_fp8(a, b, _sizes(counts), dtype)
    assert got.shape == (sum(counts), N) and got.dtype == dtype
    xs, ws = O.seen(x), [O.seen(v, 128) for v in w]
    _check_product(got, xs, ws, counts, dtype)
    assert torch.equal(got, grouped_gemm_fp8(a, b, _sizes(counts), dtype))
    if len(counts) == 1:
        assert torch.equal(got, grouped_gemm_fp8(a, b, None, dtype))
        assert torch.equal(got, grouped_gemm_fp8(a, Fp8Blocks(b.values[0], b.scales[0]), None, dtype))


def test_grouped_gemm_of_many_groups():
    g = torch.Generator().manual_seed(5)
    counts = torch.randint(0, 12, (1000,), generator=g).tolist()
    x, w = _operands(counts, 32, 48, seed=3)
    got = grouped_gemm_fp8(quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128), _sizes(counts), torch.float32)
    _check_product(got, O.seen(x), [O.seen(v, 128) for v in w], counts, torch.float32)


def test_grouped_gemm_scales_over_the_whole_range():
    """blocks whose scales lie far apart, within a row and between the operands"""
    g = torch.Generator().manual_seed(2)
    K = 640
    x = torch.randn(70, K, generator=g) * torch.exp2(torch.randint(-60, 60, (70, K // 128), generator=g).float()).repeat_interleave(128, 1)
    w = torch.randn(1, 96, K, generator=g) * torch.exp2(torch.randint(-40, 40, (1, 1, K // 128), generator=g).float()).repeat_interleave(128, 2)
    got = grouped_gemm_fp8(quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128), None, torch.float32)
    _check_product(got, O.seen(x), [O.seen(w[0], 128)], [70], torch.float32)


def test_grouped_gemm_not_a_number():
    """a NaN block reaches the results of its row, or of its 128 columns, and no others"""
    x, w = _operands([40], 300, 384)
    x[3, 200] = float("inf")
    w[0, 140, 7] = float("nan")
    got = grouped_gemm_fp8(quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128), None, torch.float32).cpu()
    expect = torch.zeros(40, 300, dtype=torch.bool)
    expect[3], expect[:, 128:256] = True, True
    assert torch.equal(got.isnan(), expect)


def test_sizes_that_do_not_fit_the_rows():
    """fewer rows than there are: the rest stays as it was; more: nothing past the last row is read or written"""
    from fma.ops.fp8.cuda_implementation import grouped_gemm_fp8_cuda

    x, w = _operands([100, 100], 64, 256)
    a, b = quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128)
    xs, ws = O.seen(x), [O.seen(v, 128) for v in w]
    out = torch.full((200, 64), 7.0, device=DEV)
    grouped_gemm_fp8_cuda(*a, *b, _sizes([60, 50]), out)
    _check_product(out, xs, ws, [60, 50], torch.float32)
    assert bool((out[110:] == 7.0).all())
    guard = torch.full((300, 64), 7.0, device=DEV)
    for sizes, counts in (([150, 4000], [150, 50]), ([-1, -1], [200, 0]), ([2**31 - 1, 2**31 - 1], [200, 0])):
        out = guard[:200].fill_(1.0)
        grouped_gemm_fp8_cuda(*a, *b, _sizes(sizes), out)
        _check_product(out, xs, ws, counts, torch.float32)
        assert bool((guard[200:] == 7.0).all())


# ---- the product with gradients --------------------------------------------------------------------------------------


def _close(got, exact, dtype, slack=0.0):
    """2-norm: half a step of the type per element, and `slack`"""
    err = float((got.cpu().double() - exact).norm() / exact.norm())
    assert err <= torch.finfo(dtype).eps / 2 + slack, err


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("counts,N,K", [([5], 16, 32), ([40, 0, 300, 7], 272, 400), ([130, 256], 512, 144)])
def test_grouped_linear(dtype, counts, N, K):
    x, w = (t.to(dtype) for t in _operands(counts, N, K, seed=K))
    dy = torch.randn(sum(counts), N, generator=torch.Generator().manual_seed(9)).to(dtype)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = grouped_linear_fp8(xd, wd, _sizes(counts))
    y.backward(dy.to(DEV))
    xs, ws, ds = O.seen(x), [O.seen(v, 128) for v in w], O.seen(dy)
    _check_product(y.detach(), xs, ws, counts, dtype)
    _check_product(xd.grad, ds, [v.t() for v in ws], counts, dtype)
    first, w_grad = 0, []
    for m in counts:
        w_grad.append(dy[first : first + m].double().t() @ xs[first : first + m])
        first += m
    # (the 16-bit form of an 8-bit value is exact in bf16; in fp16 a value under 2^-14 may lose bits, which the norm does not see)
    _close(wd.grad, torch.stack(w_grad), dtype, slack=2.0**-20)
    # one gradient at a time gives the same bits, and an input without one keeps nothing for it
    for needs in ((True, False), (False, True)):
        xa, wa = xd.detach().requires_grad_(needs[0]), wd.detach().requires_grad_(needs[1])
        grouped_linear_fp8(xa, wa, _sizes(counts)).backward(dy.to(DEV))
        assert (xa.grad is None or torch.equal(xa.grad, xd.grad)) and (wa.grad is None or torch.equal(wa.grad, wd.grad))
    with torch.no_grad():
        assert torch.equal(grouped_linear_fp8(xd, wd, _sizes(counts)), y)


def test_grouped_linear_of_no_rows():
    x, w = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16).requires_grad_(), torch.randn(2, 32, 64, device=DEV).bfloat16().requires_grad_()
    y = grouped_linear_fp8(x, w, _sizes([0, 0]))
    y.sum().backward()
    assert y.shape == (0, 32) and x.grad.shape == (0, 64) and not w.grad.any()


def test_on_another_stream_and_captured():
    """launches go to the caller's stream; a captured forward and backward pass replays on new values"""
    counts = [70, 0, 200]
    x, w = (t.bfloat16().to(DEV) for t in _operands(counts, 144, 256))
    sizes, dy = _sizes(counts), torch.randn(270, 144, device=DEV).bfloat16()
    static = x.clone()

    def step(a):
        a, b = a.detach().requires_grad_(), w.detach().requires_grad_()
        y = grouped_linear_fp8(a, b, sizes)
        return y, *torch.autograd.grad(y, (a, b), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, step(x)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for seed in range(3):
        fresh = torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(fresh)):
            assert torch.equal(a, b)
        torch.randn(1 << 20, device=DEV).sum().item()


# ---- the activation -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,I", [(1, 1), (3, 7), (2, 128), (5, 136), (9, 344), (4, 512), (33, 1408), (2, 2880)])
def test_swiglu_packed_fp8(dtype, rows, I):
    g = torch.Generator().manual_seed(rows + I)
    x = (2 * torch.randn(rows, 2 * I, generator=g) * torch.exp(torch.randn(2 * I, generator=g))).to(dtype)
    dy = torch.randn(rows, I, generator=g).to(dtype)
    xd = x.to(DEV).requires_grad_()
    y = fma.swiglu_packed_fp8(xd)
    y.backward(dy.to(DEV))
    with torch.no_grad():
        assert torch.equal(y, fma.swiglu_packed(xd)) and torch.equal(y, fma.swiglu_packed_fp8(xd))
    exact = O.swiglu_grad(O.halves(x), dy.double())
    # element by element: the arithmetic's fp32 roundings (16 of them at most; the fast sigmoid's 2 ulp in 16-bit types) and the type's own.
    # s + g s (1 - s) has no cancellation beyond a factor of 3 for |g| <= 88: its terms' magnitudes bound it.
    up, gate = O.halves(x).chunk(2, 1)
    s = torch.sigmoid(gate)
    size = torch.cat([(dy.double() * gate * s).abs(), dy.double().abs() * up.abs() * (s + gate.abs() * s * (1 - s))], 1)
    # (1 - s is formed from a rounded s: an absolute error of 2^-23, whose share is gate * s * up)
    size += torch.cat([torch.zeros_like(up), dy.double().abs() * up.abs() * gate.abs() * s], 1)
    # (the framework's sigmoid clamps its argument to +-88.376: e^-88.376 at most stands for less)
    least = 4.3e-39 * dy.double().abs() * (gate.abs() + up.abs() * (1 + 2 * gate.abs()))
    bound = 32 * 2.0**-24 * size + least.repeat(1, 2) + torch.finfo(dtype).eps / 2 * exact.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((xd.grad.cpu().double() - exact).abs() <= bound * 1.01).all())


def test_swiglu_packed_fp8_gradient_against_differences():
    """at inputs that 8 bits hold exactly the gradient is that of the activation itself"""
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-14, 15, (4, 32), generator=g).float() / 8.0  # four bits
    dy = torch.randn(4, 16, generator=g)
    xd = x.to(DEV).requires_grad_()
    fma.swiglu_packed_fp8(xd).backward(dy.to(DEV))
    step = 2.0**-12
    for i, j in ((0, 0), (1, 9), (2, 20), (3, 31)):
        d = torch.zeros_like(x, dtype=torch.float64)
        d[i, j] = step
        slope = float(((O.swiglu(x + d) - O.swiglu(x - d)) * dy.double()).sum()) / (2 * step)
        assert abs(float(xd.grad[i, j]) - slope) <= 1e-5 * max(1.0, abs(slope))


def test_swiglu_packed_fp8_keeps_half_and_takes_any_shape():
    x = torch.randn(3, 5, 2 * 1024, device=DEV).bfloat16().requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y = fma.swiglu_packed_fp8(x)
    assert y.shape == (3, 5, 1024) and sum(t.numel() * t.element_size() for t in kept) <= x.numel() * 1.02
    y.backward(torch.ones_like(y))
    rows = x.detach().view(15, 2048).requires_grad_()
    fma.swiglu_packed_fp8(rows).backward(torch.ones(15, 1024, device=DEV).bfloat16())
    assert torch.equal(x.grad.view(15, 2048), rows.grad)
    strided = torch.randn(2048, 6, device=DEV).t().requires_grad_()
    fma.swiglu_packed_fp8(strided).backward(torch.ones(6, 1024, device=DEV))
    plain = strided.detach().contiguous().requires_grad_()
    fma.swiglu_packed_fp8(plain).backward(torch.ones(6, 1024, device=DEV))
    assert torch.equal(strided.grad, plain.grad)
    empty = torch.empty(0, 64, device=DEV).requires_grad_()
    fma.swiglu_packed_fp8(empty).sum().backward()
    assert empty.grad.shape == (0, 64)
