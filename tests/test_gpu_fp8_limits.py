"""The 8-bit operators at the ends of their ranges, and what a user of them meets there: largest numbers, sizes that do not fit the rows, very many
rows, weights laid out anew behind a captured graph, the sums that a few tokens' activations are made of."""

import pytest
import torch

from fma import quantize_expert_weights, swiglu_experts_fp8
from gpu_util import DEV
from oracle import fp8_oracle as O
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
