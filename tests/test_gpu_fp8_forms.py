"""The 8-bit products in the forms and at the sizes that their other tests do not reach: tall tiles, many groups, operands past 4 GB, several
numbers of rows per group around the choice between the kernels, other streams, strided inputs, two calls at once."""

import pytest
import torch

from fma import (
    Fp8Blocks, KernelBackend, MoE, dequantize_fp8, grouped_gemm_fp8, grouped_linear_fp8, quantize_expert_weights, quantize_fp8,
    swiglu_experts_fp8, swiglu_packed, swiglu_packed_fp8,
)  # fmt: skip
from gpu_util import DEV
from oracle import fp8_oracle as O
from test_gpu_fp8 import _check_product, _operands, _sizes
from test_gpu_fp8_experts import _case, _close, _oracle

pytestmark = pytest.mark.gpu


def _random_blocks(rows, K, block_rows, seed):
    """finite e4m3 values of either sign, scales around one"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    values = torch.randint(0, 0x60, (*rows, K), generator=g, device=DEV, dtype=torch.uint8)
    values |= torch.randint(0, 2, values.shape, generator=g, device=DEV, dtype=torch.uint8) << 7
    n = 4 * ((K + 511) // 512)
    scale_rows = (*rows[:-1], (rows[-1] + block_rows - 1) // block_rows)
    scales = torch.randint(120, 132, (*scale_rows, n), generator=g, device=DEV, dtype=torch.uint8)
    return Fp8Blocks(values.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))


# 130 groups of 260 rows: tiles of 256 rows make 260 of two columns' tiles per column, more rounds of 256 compute units than tall ones
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,K", [(512, 256), (520, 144)])
def test_tall_tiles(dtype, N, K):
    counts = [260] * 129 + [288]
    x, w = _operands(counts, N, K, seed=1)
    a, b = quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128)
    got = grouped_gemm_fp8(a, b, _sizes(counts), dtype)
    some = [0, 63, 128, 129]
    rows = torch.cat([torch.arange(260 * e, 260 * e + counts[e]) for e in some])
    _check_product(got.cpu()[rows], O.seen(x[rows]), [O.seen(w[e], 128) for e in some], [counts[e] for e in some], dtype)
    # a group's sums do not depend on the tiles
    for e in range(0, 130, 7):
        rows = slice(260 * e, 260 * e + counts[e])
        alone = grouped_gemm_fp8(Fp8Blocks(a.values[rows], a.scales[rows]), Fp8Blocks(b.values[e], b.scales[e]), None, dtype)
        assert torch.equal(got[rows], alone), e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_experts_with_tall_tiles(dtype):
    E, rows, H, I = 130, 260, 256, 256
    x, gates, _, w1, w2, dy = _case(E * rows, H, I, E, 1, dtype, seed=2)
    ids = torch.arange(E * rows)[:, None] % E
    leaves = [t.to(DEV).requires_grad_() for t in (x, gates, w1, w2)]
    y = swiglu_experts_fp8(leaves[0], leaves[1], ids.to(DEV), *leaves[2:])
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    with torch.no_grad():
        served = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), w1.to(DEV), w2.to(DEV))
    for e in (0, 57, 129):
        mine = (ids[:, 0] == e).nonzero()[:, 0]
        part = [x[mine], gates[mine], w1[e : e + 1], w2[e : e + 1]]
        exact = _oracle(part[0], part[1], torch.zeros_like(ids[mine]), *part[2:], dy[mine])
        _close(y[mine.to(DEV)], exact[0], dtype, 1, "y")
        _close(served[mine.to(DEV)], exact[0], dtype, 1, "served")
        _close(grads[0][mine.to(DEV)], exact[1], dtype, 2, "dx")
        _close(grads[2][e : e + 1], exact[3], dtype, 1, "dw1")
        _close(grads[3][e : e + 1], exact[4], dtype, 1, "dw2")
        alone = [t.to(DEV).requires_grad_() for t in part]
        again = swiglu_experts_fp8(alone[0], alone[1], torch.zeros_like(ids[mine]).to(DEV), *alone[2:])
        assert torch.equal(again, y[mine.to(DEV)])
        assert torch.equal(torch.autograd.grad(again, alone[0], dy[mine].to(DEV))[0], grads[0][mine.to(DEV)])


@pytest.mark.parametrize("T", [400, 3000])
def test_experts_of_more_groups_than_a_tall_launch_has(T):
    x, gates, ids, w1, w2, dy = _case(T, 64, 48, 300, 2, torch.bfloat16, seed=3)
    exact = _oracle(x, gates, ids, w1, w2, dy)
    leaves = [t.to(DEV).requires_grad_() for t in (x, gates, w1, w2)]
    y = swiglu_experts_fp8(leaves[0], leaves[1], ids.to(DEV), *leaves[2:])
    y.backward(dy.to(DEV))
    _close(y, exact[0], torch.bfloat16, 1, "y")
    for leaf, want, links, what in zip(leaves, exact[1:], (2, 1, 1, 1), ("dx", "dgates", "dw1", "dw2")):
        _close(leaf.grad, want, torch.bfloat16, links, what)
    with torch.no_grad():
        _close(swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), *quantize_expert_weights(w1.to(DEV), w2.to(DEV))), exact[0], torch.bfloat16, 1, "served")


@pytest.mark.parametrize("N,K", [(40, 2048), (33, 144), (256, 128), (1000, 528)])
@pytest.mark.parametrize("rows", [1, 4, 8, 12, 16, 17, 25, 32, 33, 48])
def test_rows_per_group_around_the_choice_of_kernel(rows, N, K):
    counts = [rows, 0, rows + 3, max(0, rows - 5), 2 * rows, 1, rows, 0]
    x, w = _operands(counts, N, K, seed=rows)
    got = grouped_gemm_fp8(quantize_fp8(x.to(DEV)), quantize_fp8(w.to(DEV), 128), _sizes(counts), torch.float32)
    _check_product(got, O.seen(x), [O.seen(v, 128) for v in w], counts, torch.float32)


@pytest.mark.parametrize("T", [1, 2, 7, 16, 33, 64, 100])
def test_experts_around_the_choice_of_kernel(T):
    x, gates, ids, w1, w2, _ = _case(T, 272, 400, 8, 3, torch.bfloat16, seed=T)
    with torch.no_grad():
        got = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), *quantize_expert_weights(w1.to(DEV), w2.to(DEV)))
    _close(got, _oracle(x, gates, ids, w1, w2)[0], torch.bfloat16, 1, "y")


@pytest.mark.parametrize("rows", [3, 300])
def test_weights_past_4_gb(rows):
    E, N, K = 5, 32768, 32768
    b = _random_blocks((E, N), K, 128, 1)
    a = _random_blocks((E * rows,), K, 1, 2)
    got = grouped_gemm_fp8(a, b, _sizes([rows] * E), torch.float32)
    for e in (0, 4):
        mine = slice(e * rows, (e + 1) * rows)
        part = Fp8Blocks(a.values[mine], a.scales[mine])
        cut = Fp8Blocks(b.values[e, -256:].clone(), b.scales[e, -2:].clone())
        want = grouped_gemm_fp8(part, cut, None, torch.float32)  # (a few rows: in other parts of the sum)
        assert float((got[mine, -256:] - want).norm() / want.norm()) <= 2.0**-12, e


def test_rows_and_results_past_4_gb():
    R, N, K = 70000, 32768, 128
    a, b = _random_blocks((R,), K, 1, 3), _random_blocks((N,), K, 128, 4)
    got = grouped_gemm_fp8(a, b, None, torch.bfloat16)
    assert torch.equal(got[-700:], grouped_gemm_fp8(Fp8Blocks(a.values[-700:], a.scales[-700:]), b, None, torch.bfloat16))
    assert torch.equal(got[:700], grouped_gemm_fp8(Fp8Blocks(a.values[:700], a.scales[:700]), b, None, torch.bfloat16))


@pytest.mark.parametrize("T", [6, 300])
def test_strides_and_another_stream(T):
    x, gates, ids, w1, w2, dy = (t.to(DEV) for t in _case(T, 128, 144, 4, 2, torch.bfloat16, seed=5))
    leaves = [t.clone().requires_grad_() for t in (x, gates, w1, w2)]
    y = swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:])
    want = (y, *torch.autograd.grad(y, leaves, dy))
    torch.cuda.synchronize()
    wide = torch.zeros(T, 200, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:131] = x
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [wide[:, 3:131], gates.t().contiguous().t(), w1.transpose(1, 2).contiguous().transpose(1, 2), w2.clone()]
        leaves = [t.detach().requires_grad_() for t in leaves]
        y = swiglu_experts_fp8(leaves[0], leaves[1], ids.t().contiguous().t(), *leaves[2:])
        got = (y, *torch.autograd.grad(y, leaves, dy.t().contiguous().t()))
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_broadcast_gradient():
    x, gates, ids, w1, w2, _ = (t.to(DEV) for t in _case(40, 128, 144, 4, 2, torch.bfloat16, seed=6))
    one = torch.ones(40, 128, device=DEV, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, gates, w1, w2)]
    want = torch.autograd.grad(swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:]), leaves, one)
    got = torch.autograd.grad(swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:]).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    counts = _sizes([15, 0, 20, 5])
    w = torch.randn(4, 64, 128, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    want = torch.autograd.grad(grouped_linear_fp8(x, w, counts), (x, w), one[:, :64].contiguous())
    got = torch.autograd.grad(grouped_linear_fp8(x, w, counts).sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once():
    """on two streams, each with workspaces of its own"""
    cases = [[t.to(DEV) for t in _case(T, 512, 384, 8, 2, torch.bfloat16, seed=T)] for T in (700, 650)]

    def step(x, gates, ids, w1, w2, dy):
        leaves = [t.detach().requires_grad_() for t in (x, gates, w1, w2)]
        y = swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:])
        return (y, *torch.autograd.grad(y, leaves, dy))

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(3):
        for n, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[n].append(step(*c))
    torch.cuda.synchronize()
    for runs, exact in zip(got, want):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, exact))


def test_a_second_backward_reads_what_the_first_read():
    x, gates, ids, w1, w2, dy = (t.to(DEV) for t in _case(300, 256, 144, 4, 2, torch.bfloat16, seed=7))
    leaves = [t.requires_grad_() for t in (x, gates, w1, w2)]
    y = swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:])
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, dy)))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_training_step_keeps_what_is_not_a_number_to_its_token(value):
    x, gates, ids, w1, w2, dy = (t.to(DEV) for t in _case(300, 272, 144, 4, 2, torch.bfloat16, seed=8))

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, gates, w1, w2)]
        y = swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:])
        return (y, *torch.autograd.grad(y, leaves, dy))

    fine, bad = step(x), x.clone()
    bad[17, 3] = value
    got = step(bad)
    rest = torch.arange(300, device=DEV) != 17
    assert got[0][17].isnan().all() and got[1][17].isnan().all() and got[2][17].isnan().all()
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got[:3], fine[:3]))
    for a, b in zip(got[3:], fine[3:]):
        for e in range(4):
            if not (ids[17] == e).any():
                assert torch.equal(a[e], b[e]), e


def test_tokens_of_very_different_sizes():
    """a scale per token, over sixty powers of two: with every token's result brought to the same size, the norm over all of them is what it
    is for tokens of one size (a bound per token would not hold: one rounding that falls to the other side of a border is an eighth of one of
    a token's 144 activations, and the largest may carry most of the token)"""
    x, gates, ids, w1, w2, _ = _case(300, 256, 144, 4, 2, torch.bfloat16, seed=9)
    powers = torch.randint(-40, 20, (300, 1), generator=torch.Generator().manual_seed(9)).float()
    x = (x.float() * torch.exp2(powers)).bfloat16()
    exact = _oracle(x, gates, ids, w1, w2)[0]
    leaf = w1.to(DEV).requires_grad_()  # (as a training step, then as a serving one)
    trained = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), leaf, w2.to(DEV)).detach()
    with torch.no_grad():
        served = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), leaf, w2.to(DEV))
    size = exact.norm(dim=1, keepdim=True)
    for out in (trained, served):
        _close(out.cpu().double() / size, exact / size, torch.bfloat16, 1, "y")


@pytest.mark.parametrize("K", [128, 130])
def test_the_largest_float16_numbers_stay_finite(K):
    x = torch.tensor([65504.0, -65504.0, 63488.0, 63456.0, -1.0, 0.0]).half()[:, None].expand(6, K).contiguous().to(DEV)
    back = dequantize_fp8(quantize_fp8(x), torch.float16)
    assert back.isfinite().all() and bool(((back.double() - x.double()).abs() <= 2.0**-4 * x.double().abs()).all())
    wide = dequantize_fp8(quantize_fp8(x), torch.float32)
    assert float(wide[0, 0]) == 65536.0 and float(back[0, 0]) == 65504.0 and float(back[1, K - 1]) == -65504.0
    x[0, 0] = float("inf")
    assert dequantize_fp8(quantize_fp8(x), torch.float16)[0, :128].isnan().all()
    if K % 16 == 0:
        tokens = torch.full((40, K), 65504.0, device=DEV).half()
        w = (1e-6 * torch.ones(1, 32, K, device=DEV)).half().requires_grad_()
        y = grouped_linear_fp8(tokens, w, _sizes([40]))
        grad = torch.autograd.grad(y, w, torch.full_like(y, 0.015625))[0]
        assert bool(((grad.float() - 40 * 65504 * 0.015625).abs() <= 40 * 65504 * 0.015625 * 2.0**-10).all())


def _same(got, want):
    return all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(got, want, strict=True))


def test_compiled_operators():
    x, gates, ids, w1, w2, dy = (t.to(DEV) for t in _case(60, 128, 144, 8, 2, torch.bfloat16, seed=10))
    counts, blocks = _sizes([10, 0, 30, 20, 0, 0, 0, 0]), quantize_expert_weights(w1, w2)

    def conversions(x, w):
        rows, (tiles, turned) = quantize_fp8(x), quantize_fp8(w, 128, transposed=True)
        return (*rows, *tiles, *turned, dequantize_fp8(rows), dequantize_fp8(turned), grouped_gemm_fp8(rows, turned, counts))

    def serve(x, gates, ids):
        return (swiglu_experts_fp8(x, gates, ids, *blocks),)

    with torch.no_grad():
        assert _same(torch.compile(conversions, fullgraph=True)(x, w2), conversions(x, w2))
        assert _same(torch.compile(serve, fullgraph=True)(x, gates, ids), serve(x, gates, ids))

    def linear(x, w):
        return grouped_linear_fp8(x, w, counts)

    def experts(x, gates, w1, w2):
        return swiglu_experts_fp8(x, gates, ids, w1, w2)

    for call, operands in ((swiglu_packed_fp8, [x]), (linear, [x, w1]), (experts, [x, gates, w1, w2])):
        results = []
        for f in (call, torch.compile(call, fullgraph=True)):
            leaves = [t.clone().requires_grad_() for t in operands]
            y = f(*leaves)
            results.append((y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))))
        assert _same(*results), call


def test_compiled_layer():
    torch.manual_seed(0)
    moe = MoE(8, 2, 128, 144, swiglu_packed, True, False, 0.02).to(torch.bfloat16).to(DEV)
    moe.fp8_experts = True
    x = torch.randn(60, 128, device=DEV).bfloat16()

    def run(x):
        return moe(x, kernel_backend=KernelBackend.cuda)[0]

    compiled = torch.compile(run, fullgraph=True)
    grads = []
    for call in (run, compiled):
        leaf = x.clone().requires_grad_()
        y = call(leaf)
        grads.append((y.detach(), *torch.autograd.grad(y.float().pow(2).sum(), [leaf, moe.c_fc.weight, moe.c_proj.weight])))
    for a, b in zip(*grads):
        assert float((a - b).float().norm() / a.float().norm()) <= 2.0**-6  # (the traced layer's router is another kernel)
    moe.quantize_experts()
    with torch.no_grad():
        want, got = run(x), torch.compile(run, fullgraph=True)(x)
    assert float((want - got).float().norm() / want.float().norm()) <= 2.0**-6
