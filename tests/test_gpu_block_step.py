"""A training step of blocks with a norm on either side of their MoE layer, as the operators are used together: norms, router and experts, the
losses on the router's logits, the backward pass through all of them, the gradients' norm and their clipping. Against the same computed in
64 bits on the host, captured and replayed, and compiled.

Tolerance against 64 bits: a value is a chain of some twenty sums of up to 192 products in float32, each off by up to 200 units of 2^-24 of its
terms, whose magnitudes are up to a few times their sum's: 2^14 units, relative to the largest of a tensor."""

import pytest
import torch

import fma
from fma import KernelBackend, MoE, swiglu_packed
from oracle import moe_oracle as O

from gpu_util import DEV

pytestmark = pytest.mark.gpu

E, K, H, I, EPS, SCALE = 8, 2, 64, 96, 1e-5, 0.5
_TOLERANCE = 2.0**14 * 2.0**-24


class Block(torch.nn.Module):
    """stream + scale * gate * norm(MoE(normed stream)), and the norm for the next block"""

    def __init__(self) -> None:
        super().__init__()
        self.moe = MoE(E, K, H, I, swiglu_packed, True, False, 0.2)
        self.post_weight = torch.nn.Parameter(1 + 0.1 * torch.randn(H))
        self.weight = torch.nn.Parameter(1 + 0.1 * torch.randn(H))
        self.gate = torch.nn.Parameter(0.5 + 0.1 * torch.randn(H))

    def forward(self, normed, stream, mask):
        y, logits = self.moe(normed, kernel_backend=KernelBackend.cuda)
        normed, stream = fma.fused_sandwich_rmsnorm(y, stream, self.post_weight, self.weight, EPS, self.gate, SCALE)
        balance, z, counts = self.moe.router_loss(logits, mask)
        return normed, stream, 0.01 * balance + 0.001 * z, counts


def _blocks(dtype):
    torch.manual_seed(11)
    return torch.nn.ModuleList([Block() for _ in range(2)]).to(dtype).to(DEV)


def _forward(blocks, x, mask):
    normed, stream = fma.fused_residual_add_rmsnorm(x, torch.zeros_like(x), None, EPS)
    loss, counts = 0.0, []
    for block in blocks:
        normed, stream, extra, c = block(normed, stream, mask)
        loss = loss + extra
        counts.append(c)
    return normed, stream, loss, counts


def _step(forward, blocks, x, mask, dy, bound):
    for p in blocks.parameters():
        p.grad = None
    x = x.detach().requires_grad_()
    normed, stream, loss, counts = forward(blocks, x, mask)
    torch.autograd.backward([normed, stream, loss], [dy, 0.5 * dy, torch.ones_like(loss)])
    norm = fma.clip_grad_norm_(blocks.parameters(), bound)
    return [normed.detach(), stream.detach(), loss.detach(), x.grad, norm] + [c.view(torch.int32) for c in counts] + [p.grad for p in blocks.parameters()]


def _draw(dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, dy = (torch.randn(3, 40, H, generator=g, device=DEV).to(dtype) for _ in range(2))
    mask = torch.arange(40, device=DEV) < torch.tensor([[40], [23], [1]], device=DEV)
    return x, mask, dy


def test_step_against_64_bits():
    blocks = _blocks(torch.float32)
    x, mask, dy = _draw(torch.float32)
    got = _step(_forward, blocks, x, mask, dy, 0.05)

    unit = lambda v: v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)  # noqa: E731
    wide = [{n: p.detach().double().cpu().requires_grad_() for n, p in block.named_parameters()} for block in blocks]
    x64, dy64, m = x.double().cpu().requires_grad_(), dy.double().cpu(), mask.reshape(-1).cpu()
    normed, stream, loss = unit(x64), x64, 0.0
    n = int(m.sum())
    for i, w in enumerate(wide):
        rows = normed.reshape(-1, H)
        logits = rows @ w["moe.gate.weight"].t()
        selected = torch.sort(logits.detach(), dim=1, descending=True, stable=True).indices[:, :K]
        y = O.moe_experts(rows, torch.softmax(logits.gather(1, selected), -1), selected, w["moe.c_fc.weight"], w["moe.c_proj.weight"]).view_as(x64)
        stream = stream + SCALE * w["gate"] * unit(y) * w["post_weight"]
        normed = unit(stream) * w["weight"]
        counts = torch.bincount(selected[m].reshape(-1), minlength=E)
        assert torch.equal(got[5 + i].cpu().long(), counts)
        p = torch.softmax(logits, -1)[m]
        loss = loss + 0.01 * E * (counts.double() / (n * K) * p.mean(0)).sum() + 0.001 * torch.logsumexp(logits[m], -1).square().mean()
    torch.autograd.backward([normed, stream, loss], [dy64, 0.5 * dy64, torch.ones_like(loss)])
    grads = [p.grad for w in wide for p in w.values()]
    norm = torch.sqrt(sum(g.square().sum() for g in grads))
    want = [normed.detach(), stream.detach(), loss.detach(), x64.grad, norm] + [g * min(1.0, 0.05 / (float(norm) + 1e-6)) for g in grads]
    assert float(norm) > 0.1  # (there is something to clip)
    for a, b in zip(got[:5] + got[7:], want):
        assert float((a.double().cpu() - b).abs().max()) <= _TOLERANCE * float(b.abs().max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_step_replays_from_a_captured_graph(dtype):
    blocks = _blocks(dtype)
    x, mask, dy = _draw(dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(_forward, blocks, x, mask, dy, 0.05)
    torch.cuda.current_stream().wait_stream(side)
    for p in blocks.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(_forward, blocks, x, mask, dy, 0.05)
    grads = [p.grad for p in blocks.parameters()]
    for seed in range(1, 5):
        for static, fresh in zip((x, mask, dy), _draw(dtype, seed)):
            static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        want = _step(_forward, blocks, *_draw(dtype, seed), 0.05)  # eager, between the replays
        torch.cuda.synchronize()
        for p, g in zip(blocks.parameters(), grads):
            p.grad = g
        assert all(torch.equal(a, b) for a, b in zip(replayed, want))


def test_compiled_step():
    blocks = _blocks(torch.float32)
    x, mask, dy = _draw(torch.float32)
    eager = [t.clone() for t in _step(_forward, blocks, x, mask, dy, 0.05)]
    compiled = _step(torch.compile(_forward, fullgraph=True), blocks, x, mask, dy, 0.05)
    for a, b in zip(eager, compiled):
        if a.dtype == torch.int32:
            assert torch.equal(a, b)
        else:
            assert float((a - b).abs().max()) <= _TOLERANCE * float(a.abs().max())
