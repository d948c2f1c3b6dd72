"""The 8-bit operators at the ends of their ranges, and what a user of them meets there: largest numbers, sizes that do not fit the rows, very many
rows, weights laid out anew behind a captured graph, the sums that a few tokens' activations are made of."""

import pytest
import torch

from fma import (
    KernelBackend, MoE, dequantize_fp8, grouped_linear_fp8, quantize_expert_weights, quantize_fp8,
    swiglu_experts_fp8, swiglu_packed, swiglu_packed_fp8,
)  # fmt: skip
from gpu_util import DEV
from oracle import fp8_oracle as O
from test_gpu_fp8 import _sizes
from test_gpu_fp8_experts import _case, _close, _oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k", [(40, 1), (300, 2)])
def test_activations_past_float16s_range(T, k):
    """up and gate of some 300 make activations of 90000, which the forward pass takes as they are (its sums are fp32), and so do the gradients"""
    x, gates, ids, w1, w2, dy = _case(T, 128, 144, 3, k, torch.float16, seed=T)
    I = 144
    for column in (3, 140):  # (a column of each of the two blocks)
        w1[:, column] *= 400
        w1[:, I + column] *= 400
        w2[:, :, column] *= 2.0**-10
    dy = dy * 2.0**-8  # (the weight gradient's elements stay below 65504)
    y, dx, dg, dw1, dw2 = _oracle(x, gates, ids, w1, w2, dy)
    assert float(dw2.abs().max()) < 65504 and float(y.abs().max()) < 65504
    h = O.seen(x) @ O.seen(w1[0, :I], 128).t(), O.seen(x) @ O.seen(w1[0, I:], 128).t()
    assert float((h[0] * h[1] * torch.sigmoid(h[1])).abs().max()) > 2**17
    leaves = [t.to(DEV).requires_grad_() for t in (x, gates, w1, w2)]
    got = swiglu_experts_fp8(leaves[0], leaves[1], ids.to(DEV), *leaves[2:])
    got.backward(dy.to(DEV))
    _close(got, y, torch.float16, 1, "y")
    wide = torch.zeros(I, dtype=torch.bool)
    wide[[3, 140]] = True
    both = wide.repeat(2)
    for what, a, b, links in (("dx", leaves[0].grad, dx, 2), ("dgates", leaves[1].grad, dg, 1), ("dw1 wide", leaves[2].grad[:, both], dw1[:, both], 1),
                              ("dw1", leaves[2].grad[:, ~both], dw1[:, ~both], 1), ("dw2 wide", leaves[3].grad[:, :, wide], dw2[:, :, wide], 1),
                              ("dw2", leaves[3].grad[:, :, ~wide], dw2[:, :, ~wide], 1)):  # fmt: skip
        assert bool(a.isfinite().all()), what
        _close(a, b, torch.float16, links, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [128, 130])
def test_the_largest_numbers_stay_finite(dtype, K):
    """248 * 2^120 and more is 2^128 in 8 bits, which no 16- or 32-bit number is: it comes back as the type's largest"""
    most = torch.finfo(dtype).max
    x = torch.tensor([most, -most, 248 * 2.0**120, 247 * 2.0**120, 240 * 2.0**120, -1.0]).to(dtype)[:, None].expand(6, K).contiguous()
    blocks = quantize_fp8(x.to(DEV))
    assert torch.equal(blocks.values[:3, 0].float().cpu(), torch.tensor([256.0, -256.0, 256.0]))  # (248: a tie, to the even one)
    for rows in (1, 128):
        back = dequantize_fp8(quantize_fp8(x.to(DEV), rows), dtype).cpu().double()
        assert back.isfinite().all() and float(back[0, 0]) == most == -float(back[1, K - 1])
        # half a step of e4m3, relative to the value
        assert bool(((back - x.double()).abs()[:5] <= 2.0**-4 * x.double().abs()[:5]).all())
        assert float(back[4, 0]) == 240 * 2.0**120
    x[0, 0] = float("inf")
    assert dequantize_fp8(quantize_fp8(x.to(DEV)), dtype)[0, :128].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("I", [128, 130])
def test_gradients_at_the_largest_numbers(dtype, I):
    """a gate of 2^128 in 8 bits lets everything through, and so does its slope"""
    most = torch.finfo(dtype).max
    x = torch.zeros(2, 2 * I)
    x[:, :I] = 2.0**-100  # up
    x[0, I:], x[1, I:] = most, 1.0
    leaf = x.to(dtype).to(DEV).requires_grad_()
    y = swiglu_packed_fp8(leaf)
    y.backward(torch.full_like(y, 0.5))
    assert y.isfinite().all() and leaf.grad.isfinite().all()
    # d up = gate / 2, within half a step of e4m3 and one of the type; d gate = up / 2
    assert bool(((leaf.grad[0, :I].double().cpu() / (most / 2) - 1).abs() <= 2.0**-4 + torch.finfo(dtype).eps).all())
    assert bool(((leaf.grad[0, I:].double().cpu() / 2.0**-101 - 1).abs() <= torch.finfo(dtype).eps).all())


def test_an_experts_gradient_at_the_largest_pre_activation():
    """a gate of 248 * 2^120, which is 2^128 where it is kept in 8 bits; every product on the way to the tokens' gradient is a power of two or exact"""
    x, gates, ids = torch.full((3, 128), 2.0**100).bfloat16(), torch.ones(3, 1).bfloat16(), torch.zeros(3, 1, dtype=torch.int32)
    w1 = torch.full((1, 256, 128), 2.0**-110)
    w1[:, 128:, 0::2], w1[:, 128:, 1::2] = 1.875 * 2.0**20, 2.0**21
    w1, w2, dy = w1.bfloat16(), torch.full((1, 128, 128), 2.0**-120).bfloat16(), torch.full((3, 128), 2.0**20).bfloat16()
    leaf = x.to(DEV).requires_grad_()
    y = swiglu_experts_fp8(leaf, gates.to(DEV), ids.to(DEV), w1.to(DEV), w2.to(DEV))
    y.backward(dy.to(DEV))
    assert bool((y == 128 * 32).all())  # (31 * 2^120 is 32 * 2^120 in 8 bits)
    # d up = da gate = 2^-93 2^128, d gate = da up = 2^-93 2^-3; two roundings to the type, one step of the scale
    exact = 128 * 2.0**35 * w1[0, 0].double() + 128 * 2.0**-96 * w1[0, 128].double()
    assert bool(((leaf.grad.cpu().double() - exact).abs() <= exact * (torch.finfo(torch.bfloat16).eps + 2.0**-23)).all())


def test_weight_gradient_of_the_largest_tokens():
    most = torch.finfo(torch.bfloat16).max
    tokens, w = torch.full((40, 128), most, device=DEV).bfloat16(), (1e-36 * torch.ones(1, 32, 128, device=DEV)).bfloat16().requires_grad_()
    y = grouped_linear_fp8(tokens, w, _sizes([40]))
    grad = torch.autograd.grad(y, w, torch.full_like(y, 2.0**-20))[0]
    assert bool(((grad.double() / (40 * most * 2.0**-20) - 1).abs() <= 2.0**-8 + 40 * 2.0**-23).all())


@pytest.mark.parametrize("counts,clamped", [([30, 4000], [30, 42]), ([2**31 - 1, 2**31 - 1], [72, 0]), ([-1, -1, 5], [72, 0, 0]), ([20, 10, 0], [20, 10, 0]),
                                            ([72] + [-1] * 200, [72] + [0] * 200)])  # fmt: skip
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_sizes_that_do_not_fit_the_rows(dtype, counts, clamped):
    """rows past the last one do not exist, whatever the sizes say: output and gradients are those of the sizes cut to the rows"""
    R, N, K, E = 72, 48, 64, len(counts)
    g = torch.Generator().manual_seed(E)
    x, w, dy = (torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((R, K), (E, N, K), (R, N)))
    rows = sum(clamped)
    results = []
    for sizes in (counts, clamped):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = grouped_linear_fp8(a, b, _sizes(sizes))
        x_grad, w_grad = torch.autograd.grad(y, (a, b), dy)
        results.append((y[:rows], x_grad[:rows], w_grad))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_a_layer_laid_out_anew_behind_a_captured_graph():
    """quantize_experts() after a change of the weights: a graph captured before it serves the new ones"""
    torch.manual_seed(0)
    moe = MoE(8, 2, 128, 144, swiglu_packed, True, False, 0.05).to(torch.bfloat16).to(DEV)
    moe.quantize_experts()
    x = torch.randn(12, 128, device=DEV).bfloat16()

    def run():
        return moe(x, kernel_backend=KernelBackend.cuda)[0]

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = run()
        first = run().clone()
        for seed in range(3):
            moe.c_fc.weight.copy_(0.1 * torch.randn(moe.c_fc.weight.shape, generator=torch.Generator().manual_seed(seed)))
            moe.c_proj.weight.mul_(1.5)
            before = [t.data_ptr() for b in moe._fp8_weights[1] for t in b]
            if seed == 1:
                with torch.inference_mode():  # (serving programs call it there too)
                    moe.quantize_experts()
            else:
                moe.quantize_experts()
            assert [t.data_ptr() for b in moe._fp8_weights[1] for t in b] == before
            graph.replay()
            torch.cuda.synchronize()
            want = run()
            assert torch.equal(captured, want) and not torch.equal(captured, first)
            junk = [torch.full_like(t.view(torch.uint8), 0x7E) for b in moe._fp8_weights[1] for t in b]  # (whatever was freed is overwritten)
            torch.randn(1 << 20, device=DEV).sum().item()
            del junk
        # a copy has blocks of its own
        import copy

        other = copy.deepcopy(moe).quantize_experts()
        other.c_proj.weight.mul_(2)
        other.quantize_experts()
        assert torch.equal(run(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,I,E", [(64, 1024, 512, 8), (24, 2048, 1408, 6)])
def test_a_few_tokens_hold_few_stray_roundings(dtype, T, H, I, E):
    """The activation of a few tokens is quantised from sums of exact products, as a training step's pre-activation is: a sum is off by about 2^-22 of
    itself, and an e4m3 step is 2^-3 to 2^-4 of a value wide, so that about one activation in 2^17 is rounded to the other side of a border
    (with products cut at 2^-13, as the 8-bit instruction does it, one in 2^11). A token with such an activation is off by some 2^-4 of it, a
    2^-8th of the token. Expected are 0.25 such tokens; four and more are one run in ten thousand. All others: 2^-13, for the 8-bit sums of the
    second product (2^-16, root mean square); of every element, what half a step of its type explains is left out."""
    x, gates, ids, w1, w2, _ = _case(T, H, I, E, 1, dtype, seed=T)
    exact = _oracle(x, gates, ids, w1, w2)[0]
    with torch.no_grad():
        got = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), *quantize_expert_weights(w1.to(DEV), w2.to(DEV))).cpu().double()
    # an element's rounding to the type explains half a step of it; what is left is the sum's
    left = ((got - exact).abs() - torch.finfo(dtype).eps / 2 * exact.abs()).clamp(min=0)
    off = left.norm(dim=1) / exact.norm(dim=1)
    assert int((off > 2.0**-13).sum()) <= 3, (int((off > 2.0**-13).sum()), float(off.max()))


def test_conversions_of_very_many_rows():
    """more rows than one launch of the 16-byte kernels has threads for"""
    for rows, dtype in ((2**28 + 5, torch.bfloat16), (2**27 + 5, torch.float32)):
        x = torch.randn(1 << 16, 16, device=DEV).to(dtype).repeat(rows // (1 << 16) + 1, 1)[:rows]
        values, scales = quantize_fp8(x)
        for part in (slice(0, 70000), slice(rows - 70000, rows)):
            few = quantize_fp8(x[part])
            assert torch.equal(few.values.view(torch.uint8), values[part].view(torch.uint8))
            assert torch.equal(few.scales.view(torch.uint8), scales[part].view(torch.uint8))
        del x, values, scales
    rows = 2**27 + 3
    x = torch.randn(1 << 16, 16, device=DEV).bfloat16().repeat(rows // (1 << 16) + 1, 1)[:rows].requires_grad_()
    y = swiglu_packed_fp8(x)
    y.backward(torch.ones_like(y))
    for part in (slice(0, 70000), slice(rows - 70000, rows)):
        few = x.detach()[part].requires_grad_()
        z = swiglu_packed_fp8(few)
        z.backward(torch.ones_like(z))
        assert torch.equal(y[part], z) and torch.equal(x.grad[part], few.grad)
