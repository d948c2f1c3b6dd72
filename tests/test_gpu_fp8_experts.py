"""The expert path in 8 bits against the 64-bit oracle, and the MoE layer that runs it."""

import copy

import pytest
import torch

import fma
from fma import KernelBackend, MoE, quantize_expert_weights, swiglu_experts_fp8, swiglu_packed
from gpu_util import DEV
from oracle import fp8_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _case(T, H, I, E, k, dtype, seed=0, one_expert=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(H, generator=g))).to(dtype)
    w1, w2 = (0.08 * torch.randn(E, n, m, generator=g) for n, m in ((2 * I, H), (H, I)))
    logits = torch.randn(T, E, generator=g)
    if one_expert:
        logits[:, E // 2] += 100.0
    gates, ids = logits.topk(k, dim=1)
    return x, torch.softmax(gates, 1).to(dtype), ids, w1.to(dtype), w2.to(dtype), torch.randn(T, H, generator=g).to(dtype)


def _oracle(x, gates, ids, w1, w2, dy=None):
    """(y, dx, dgates, dw1, dw2) in 64 bits"""
    T, H = x.shape
    E, two_I, _ = w1.shape
    I = two_I // 2
    xs, g = O.seen(x), gates.double()
    y, dx, dg = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64), torch.zeros_like(g)
    dw1, dw2 = torch.zeros(w1.shape, dtype=torch.float64), torch.zeros(w2.shape, dtype=torch.float64)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        s1, s2 = torch.cat([O.seen(w1[e, :I], 128), O.seen(w1[e, I:], 128)]), O.seen(w2[e], 128)
        h = xs[t] @ s1.t()
        a = O.seen(O.swiglu(h))
        o = a @ s2.t()
        y.index_add_(0, t, o * g[t, j, None])
        if dy is None:
            continue
        d = dy.double()[t]
        dg[t, j] = (d * o).sum(1)
        do = d * g[t, j, None]
        dh = O.swiglu_grad(O.halves(h), O.seen(do) @ s2)
        dx.index_add_(0, t, O.halves(dh) @ s1)
        dw1[e], dw2[e] = dh.t() @ xs[t], do.t() @ a
    return y, dx, dg, dw1, dw2


def _close(got, exact, dtype, links, what):
    """2-norm. Two roundings to the 16-bit type (half a step each), and for every quantised tensor on the way that is made from sums: a sum is
    off by about 2^-15 of itself (the 8-bit matrix instruction's cut, 2^-13 of the largest of eight products, over many of them), so
    that about one value in 2^11 falls to the other side of a border between two e4m3 steps, which lie 2^-3 to 2^-4 of a value apart:
    2^-3.5 * 2^-5.5 = 2^-9 in the norm. Four times that per link."""
    err = float((got.detach().cpu().double() - exact).norm() / exact.norm())
    assert err <= torch.finfo(dtype).eps + links * 2.0**-7, (what, err)


SIZES = [
    (1, 16, 16, 1, 1), (1, 128, 128, 4, 2), (3, 64, 48, 5, 3), (37, 256, 208, 6, 2), (70, 400, 144, 3, 3), (300, 512, 384, 4, 2),
    (40, 288, 1040, 8, 8), (129, 1024, 272, 2, 1),
]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,I,E,k", SIZES)
def test_experts(dtype, T, H, I, E, k):
    x, gates, ids, w1, w2, dy = _case(T, H, I, E, k, dtype, seed=T + H)
    y, dx, dg, dw1, dw2 = _oracle(x, gates, ids, w1, w2, dy)
    leaves = [t.to(DEV).requires_grad_() for t in (x, gates, w1, w2)]
    got = swiglu_experts_fp8(leaves[0], leaves[1], ids.to(DEV), *leaves[2:])
    got.backward(dy.to(DEV))
    _close(got, y, dtype, 1, "y")
    for leaf, exact, links, what in zip(leaves, (dx, dg, dw1, dw2), (2, 1, 1, 1), ("dx", "dgates", "dw1", "dw2")):
        assert leaf.grad.dtype == dtype
        if float(exact.norm()):
            _close(leaf.grad, exact, dtype, links, what)
    blocks = quantize_expert_weights(w1.to(DEV), w2.to(DEV))
    with torch.no_grad():
        served = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(torch.int32).to(DEV), *blocks)
        assert torch.equal(served, swiglu_experts_fp8(leaves[0], leaves[1], ids.to(DEV), *leaves[2:]))
    _close(served, y, dtype, 1, "served")
    # one gradient at a time: the same bits
    for i in range(4):
        alone = [t.detach().requires_grad_(i == n) for n, t in enumerate(leaves)]
        swiglu_experts_fp8(alone[0], alone[1], ids.to(DEV), *alone[2:]).backward(dy.to(DEV))
        assert torch.equal(alone[i].grad, leaves[i].grad) and all(t.grad is None for n, t in enumerate(alone) if n != i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,I,E,k", [(192, 1024, 384, 16, 2), (160, 2048, 256, 1, 1), (300, 512, 512, 1, 1)])
def test_weight_gradients_hold_no_stray_roundings(dtype, T, H, I, E, k):
    """Element by element, where the norm hides single ones. The pre-activation is summed to fp32, so that a sum is off by about 2^-22 of
    itself, and an e4m3 step is 2^-3 to 2^-4 of a value wide: of 2^17 values about one is rounded to the other side of a border, and with it
    a row of an expert's up-projection gradient is off. One in 2^15 is allowed. (With products cut at 2^-13, as the 8-bit instruction does it,
    sums are off by 2^-16: 49, 13 and 18 rows are visibly off in float16 where the oracle's sums are perturbed by that.)
    Of a row not hit, an element is off by two roundings to the type, by the 8-bit cut of the gradient's sum (2^-15) and by fp32 sums: below
    eps + 2^-12; eight times that counts as off."""
    x, gates, ids, w1, w2, dy = _case(T, H, I, E, k, dtype, seed=T)
    dw1 = _oracle(x, gates, ids, w1, w2, dy)[3]
    leaf = w1.to(DEV).requires_grad_()
    swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), leaf, w2.to(DEV)).backward(dy.to(DEV))
    off = (leaf.grad.cpu().double() - dw1).abs() / dw1.abs().clamp(min=float(dw1.pow(2).mean().sqrt()))
    stray = (off > 8 * (torch.finfo(dtype).eps + 2.0**-12)).any(-1)
    assert int(stray.sum()) <= T * k * 2 * I // 2**15, (int(stray.sum()), float(off.max()))


def test_every_token_with_the_same_expert():
    x, gates, ids, w1, w2, dy = _case(700, 256, 128, 8, 2, torch.bfloat16, one_expert=True)
    y, dx, *_ = _oracle(x, gates, ids, w1, w2, dy)
    leaf = x.to(DEV).requires_grad_()
    got = swiglu_experts_fp8(leaf, gates.to(DEV), ids.to(DEV), w1.to(DEV), w2.to(DEV))
    got.backward(dy.to(DEV))
    _close(got, y, torch.bfloat16, 1, "y")
    _close(leaf.grad, dx, torch.bfloat16, 2, "dx")


@pytest.mark.parametrize("T", [5, 300])
def test_choices_that_name_no_expert(T):
    """they contribute nothing, and their gates have no gradient"""
    x, gates, ids, w1, w2, dy = _case(T, 128, 128, 4, 3, torch.bfloat16, seed=1)
    ids[0, 0], ids[T - 1, 2], ids[2] = -1, 4, 1 << 20
    y, dx, dg, dw1, dw2 = _oracle(x, gates, ids, w1, w2, dy)
    for kind in (torch.int32, torch.int64):
        leaves = [t.to(DEV).requires_grad_() for t in (x, gates, w1, w2)]
        got = swiglu_experts_fp8(leaves[0], leaves[1], ids.to(kind).to(DEV), *leaves[2:])
        got.backward(dy.to(DEV))
        assert not got[2].any() and not leaves[0].grad[2].any() and not leaves[1].grad[2].any()
        assert float(leaves[1].grad[0, 0]) == 0.0 == float(leaves[1].grad[T - 1, 2])
        _close(got, y, torch.bfloat16, 1, "y")
        for leaf, exact, links, what in zip(leaves, (dx, dg, dw1, dw2), (2, 1, 1, 1), ("dx", "dgates", "dw1", "dw2")):
            _close(leaf.grad, exact, torch.bfloat16, links, what)
        with torch.no_grad():
            served = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(kind).to(DEV), *quantize_expert_weights(w1.to(DEV), w2.to(DEV)))
        assert not served[2].any()
        _close(served, y, torch.bfloat16, 1, "served")


def test_no_tokens():
    x, gates, ids, w1, w2, _ = _case(4, 64, 32, 3, 2, torch.bfloat16)
    leaves = [t.to(DEV).requires_grad_() for t in (x[:0], gates[:0], w1, w2)]
    y = swiglu_experts_fp8(leaves[0], leaves[1], ids[:0].to(DEV), *leaves[2:])
    y.sum().backward()
    assert y.shape == (0, 64) and all(t.grad.shape == t.shape for t in leaves) and not leaves[2].grad.any() and not leaves[3].grad.any()


def test_a_token_that_is_not_a_number_stays_alone():
    x, gates, ids, w1, w2, _ = _case(300, 256, 128, 4, 2, torch.bfloat16)
    with torch.no_grad():
        fine = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), w1.to(DEV), w2.to(DEV))
        x[17, 3] = float("inf")
        got = swiglu_experts_fp8(x.to(DEV), gates.to(DEV), ids.to(DEV), w1.to(DEV), w2.to(DEV))
    assert got[17].isnan().all()
    rest = torch.arange(300, device=DEV) != 17
    assert torch.equal(got[rest], fine[rest])


@pytest.mark.parametrize("T", [1, 9, 270])
def test_captured(T):
    """a serving step and a training step replay on new tokens and routings"""
    x, gates, ids, w1, w2, dy = (t.to(DEV) for t in _case(T, 256, 384, 6, 2, torch.bfloat16))
    blocks = quantize_expert_weights(w1, w2)
    static = [x.clone(), gates.clone(), ids.clone()]

    def serve(x, gates, ids):
        with torch.no_grad():
            return (swiglu_experts_fp8(x, gates, ids, *blocks),)

    def train(x, gates, ids):
        leaves = [t.detach().requires_grad_() for t in (x, gates, w1, w2)]
        y = swiglu_experts_fp8(leaves[0], leaves[1], ids, *leaves[2:])
        return (y, *torch.autograd.grad(y, leaves, dy))

    for step in (serve, train):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step(*static)
        for seed in (1, 2, 3):
            fresh = [t.to(DEV) for t in _case(T, 256, 384, 6, 2, torch.bfloat16, seed=seed)[:3]]
            for s, f in zip(static, fresh):
                s.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(captured, step(*fresh)):
                assert torch.equal(a, b)
            torch.randn(1 << 20, device=DEV).sum().item()


# ---- the layer ------------------------------------------------------------------------------------------------------


def _layer(dtype=torch.bfloat16, H=256, I=384, E=8, k=2, **kwargs):
    torch.manual_seed(3)
    return MoE(E, k, H, I, swiglu_packed, True, kwargs.pop("bias", False), 0.05).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 40, 500])
def test_layer(dtype, T):
    moe = _layer(dtype)
    x = torch.randn(T, 256, generator=torch.Generator().manual_seed(T)).to(dtype).to(DEV)
    with torch.no_grad():
        sixteen, logits16 = moe(x, kernel_backend=KernelBackend.cuda)
    moe.fp8_experts = True
    leaf = x.detach().requires_grad_()
    y, logits = moe(leaf, kernel_backend=KernelBackend.cuda)
    y.square().sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in moe.parameters()) and leaf.grad is not None
    logits16_, gates, ids = moe._compute_routing_weights(x)
    exact = _oracle(x.cpu(), gates.detach().cpu(), ids.cpu(), moe.c_fc.weight.detach().cpu(), moe.c_proj.weight.detach().cpu())[0]
    _close(y, exact, dtype, 1, "y")
    with torch.no_grad():
        alone = moe(x, kernel_backend=KernelBackend.cuda)[0]  # (no backward follows: another kernel for few tokens)
        _close(alone, exact, dtype, 1, "alone")
        served = moe.quantize_experts()(x, kernel_backend=KernelBackend.cuda)[0]
        assert torch.equal(served, alone)
        # 8-bit products against 16-bit ones: three quantised operands on the way, each off by 2^-5.2 of itself in the norm (uniform
        # within half a step of 2^-3 .. 2^-4), and twice that
        assert float((served - sixteen).float().norm() / sixteen.float().norm()) <= 2 * 5**0.5 * 2.0**-5.2
        # weights that have changed since are used as they are
        moe.c_proj.weight.mul_(2)
        assert torch.allclose(moe(x, kernel_backend=KernelBackend.cuda)[0].float(), 2 * alone.float(), rtol=2.0**-7, atol=1e-3)
        assert torch.equal(moe.quantize_experts()(x, kernel_backend=KernelBackend.cuda)[0], moe(x, kernel_backend=KernelBackend.cuda)[0])
    other = copy.deepcopy(moe)
    with torch.no_grad():
        assert torch.equal(other(x, kernel_backend=KernelBackend.cuda)[0], moe(x, kernel_backend=KernelBackend.cuda)[0])


def test_layer_refusals():
    x = torch.randn(4, 256, device=DEV).bfloat16()
    biased = _layer(bias=True)
    biased.fp8_experts = True
    with pytest.raises(ValueError, match="biases"):
        biased(x, kernel_backend=KernelBackend.cuda)
    with pytest.raises(ValueError, match="biases"):
        biased.quantize_experts()
    single = _layer(torch.float32)
    single.fp8_experts = True
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        single(x.float(), kernel_backend=KernelBackend.cuda)
    odd = _layer(I=24)
    odd.fp8_experts = True
    with pytest.raises(ValueError, match="multiples of 16"):
        odd(x, kernel_backend=KernelBackend.cuda)
    gelu = MoE(4, 2, 256, 384, torch.nn.functional.gelu, False, False, 0.02).to(torch.bfloat16).to(DEV)
    gelu.fp8_experts = True
    with pytest.raises(ValueError, match="swiglu_packed"):
        gelu(x, kernel_backend=KernelBackend.cuda)


def test_layer_with_the_activation_kept_in_8_bits():
    """swiglu_packed_fp8 as a layer's activation: the 16-bit layer with less memory between forward and backward"""
    torch.manual_seed(0)
    moe = MoE(4, 2, 128, 256, fma.swiglu_packed_fp8, True, False, 0.05).to(torch.bfloat16).to(DEV)
    same = MoE(4, 2, 128, 256, swiglu_packed, True, False, 0.05).to(torch.bfloat16).to(DEV)
    same.load_state_dict(moe.state_dict())
    x = torch.randn(90, 128, device=DEV).bfloat16()
    a, b = x.detach().requires_grad_(), x.detach().requires_grad_()
    ya, yb = moe(a, kernel_backend=KernelBackend.cuda)[0], same(b, kernel_backend=KernelBackend.cuda)[0]
    assert torch.equal(ya, yb)
    dy = torch.randn_like(ya)
    ya.backward(dy)
    yb.backward(dy)
    # the gradient at values that are off by 2^-5.2 of themselves in the norm; its slope in them is of the order of one
    assert float((a.grad - b.grad).float().norm() / b.grad.float().norm()) <= 4 * 2.0**-5.2
    assert torch.equal(moe.c_proj.weight.grad, same.c_proj.weight.grad)
