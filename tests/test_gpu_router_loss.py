"""router_loss against its formulas in 64 bits.

Tolerances, with u = 2^-24, x = logit - largest logit of the token and X = sum_e p_e |x_e|: an exponential is off by (3 |x| + 4) u (its argument
rounded twice, the function to two units), a token's sum by what its terms are and 16 additions, a probability by rel = (3 |x| + 3 X + 40) u,
the log of the sum by (3 X + 24) u and two roundings of its parts. A lane adds at most T / 256 + 1 probabilities in float32 one after the
other, six additions join the lanes and sixteen the wavefronts; from there on 64 bits. A gradient has six more roundings, and the one to its type."""

import pytest
import torch

import fma
from fma import MoE, swiglu_packed

from gpu_util import DEV

pytestmark = pytest.mark.gpu

_U = 2.0**-24
_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}  # half of the smallest number


def _exact(logits, k, mask, gb, gz):
    """values and bounds in 64 bits; logits [T, E] finite in the rows that count"""
    l64 = logits.detach().double()
    T, E = l64.shape
    keep = torch.ones(T, dtype=torch.bool, device=DEV) if mask is None else mask.reshape(-1)
    rows = l64[keep]
    n = max(1, rows.shape[0])
    top = rows.amax(1, keepdim=True) if rows.shape[0] else rows[:, :1]
    x = rows - top
    sums = torch.exp(x).sum(1, keepdim=True)
    p, lse = torch.exp(x) / sums, top + torch.log(sums)
    # places by a stable sort of the negated logits: the lowest expert first among equal ones
    chosen = torch.sort(rows, dim=1, descending=True, stable=True).indices[:, :k]
    counts = torch.bincount(chosen.reshape(-1), minlength=E)
    f = counts.double() / (n * k)
    big_x = (p * x.abs()).sum(1, keepdim=True)
    rel = (3 * x.abs() + 3 * big_x + 40) * _U
    lse_err = (3 * big_x + 24) * _U + 2 * _U * (top.abs() + torch.log(sums).abs())
    balance, z = E * (f * p.sum(0)).sum() / n, (lse * lse).sum() / n
    balance_bound = E * (f * (p * rel).sum(0)).sum() / n + (T / 256 + 32) * _U * balance
    z_bound = (2 * lse.abs() * lse_err).sum() / n + 4 * _U * z
    s = E * (p * f).sum(1, keepdim=True)
    grad = (gb * p * (E * f - s) + 2 * gz * lse * p) / n
    bound = abs(gb) * ((E * f + s) * (rel + 8 * _U) + E * (p * f * rel).sum(1, keepdim=True)) + 2 * abs(gz) * (lse.abs() * (rel + 8 * _U) + lse_err)
    bound = bound * p / n * (1 + 2.0**-10) + grad.abs() * torch.finfo(logits.dtype).eps / 2 * (1 + 2.0**-10) + _TINY[logits.dtype]
    bound = bound + 2.0**-126 * (abs(gb) * E + 2 * abs(gz) * lse.abs()) / n  # (an exponential below the normal numbers may be zero)
    full, full_bound = torch.zeros_like(l64), torch.zeros_like(l64)
    full[keep], full_bound[keep] = grad, bound
    return (balance, balance_bound), (z, z_bound), counts, (full, full_bound)


def _run(logits, k, mask, gb, gz):
    leaf = logits.detach().requires_grad_()
    balance, z, counts = fma.router_loss(leaf, k, mask)
    assert balance.dtype == z.dtype == torch.float32 and balance.shape == z.shape == () and counts.dtype == torch.uint32
    grads = [torch.tensor(g, device=DEV) for g in (gb, gz)]
    torch.autograd.backward([balance, z], grads)
    return balance.detach(), z.detach(), counts, leaf.grad


def _check(logits, k, mask=None, gb=0.7, gz=-0.3, got=None):
    balance, z, counts, grad = got or _run(logits, k, mask, gb, gz)
    want = _exact(logits.reshape(-1, logits.shape[-1]), k, mask, gb, gz)
    assert torch.equal(counts.view(torch.int32).long(), want[2])
    for value, (exact, bound) in zip((balance, z), want[:2]):
        assert abs(float(value) - float(exact)) <= float(bound), (float(value), float(exact), float(bound))
    assert grad.shape == logits.shape and grad.dtype == logits.dtype
    assert bool(((grad.double().reshape(want[3][0].shape) - want[3][0]).abs() <= want[3][1]).all())


def _logits(T, E, dtype, seed=0, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * E + T)
    return (spread * torch.randn(T, E, generator=g, device=DEV)).to(dtype)


# every number of lanes per token (1 to 64) and both numbers of logits per lane, its ends, rows that are no whole vectors
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("E", [1, 2, 3, 7, 8, 9, 16, 17, 31, 32, 40, 60, 64, 65, 128, 129, 200, 256, 257, 500, 512, 513, 1000, 1024])
def test_against_fp64(E, dtype):
    for T in (1, 5, 130, 1001):
        for k in sorted({1, min(2, E), min(8, E), E}):
            _check(_logits(T, E, _DTYPES[dtype]), k)


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("E,k", [(8, 2), (64, 8), (128, 5), (1000, 8)])
def test_equal_logits(E, k, dtype):
    """logits of a few values, rows of one value, both zeros: the lowest experts come first"""
    g = torch.Generator(device=DEV).manual_seed(E)
    logits = torch.randint(-2, 3, (777, E), generator=g, device=DEV).to(_DTYPES[dtype])
    logits[5] = 1.5
    logits[6] = -0.0
    logits[6, E // 2 :] = 0.0
    logits[7, :] = 0.0
    logits[7, : E // 2] = -0.0
    _check(logits, k)
    counts = fma.router_loss(logits[5:8], k)[2].view(torch.int32)
    assert counts.tolist() == [3] * k + [0] * (E - k)


@pytest.mark.parametrize("dtype", _DTYPES)
def test_close_logits(dtype):
    """neighbouring numbers of the type: the choice turns on the last bit"""
    start = torch.tensor(1.0, dtype=_DTYPES[dtype], device=DEV)
    ints = {4: torch.int32, 2: torch.int16}[start.element_size()]
    steps = torch.stack([torch.randperm(64, generator=torch.Generator().manual_seed(i)) for i in range(300)]).to(DEV).to(ints)
    _check((start.view(ints) + steps).view(_DTYPES[dtype]), 8)
    _check(-(start.view(ints) + steps).view(_DTYPES[dtype]), 8)


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("T,E,k", [(40000, 64, 8), (70001, 8, 2), (20011, 256, 4), (3001, 1024, 8)])
def test_many_tokens_and_a_mask(T, E, k, dtype):
    logits = _logits(T, E, _DTYPES[dtype])
    mask = torch.rand(T, generator=torch.Generator(device=DEV).manual_seed(T), device=DEV) < 0.6
    _check(logits, k)
    first = _run(logits, k, mask, 1.0, 1.0)
    _check(logits, k, mask, 1.0, 1.0, first)
    again = _run(logits, k, mask, 1.0, 1.0)
    assert all(torch.equal(a.view(torch.int32) if a.dtype == torch.uint32 else a, b.view(torch.int32) if b.dtype == torch.uint32 else b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("E", [8, 60, 128, 1024])
def test_what_masked_tokens_hold_does_not_matter(E, dtype):
    logits = _logits(300, E, _DTYPES[dtype])
    mask = torch.ones(300, dtype=torch.bool, device=DEV)
    mask[::3] = False
    want = _run(logits, 2, mask, 1.0, 1.0)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(logits.dtype).min):
        logits[::3] = bad
        got = _run(logits, 2, mask, 1.0, 1.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2].view(torch.int32), want[2].view(torch.int32))
        assert torch.equal(got[3], want[3]) and not got[3][::3].any()


@pytest.mark.parametrize("dtype", _DTYPES)
def test_nothing_counts(dtype):
    logits = _logits(100, 16, _DTYPES[dtype])
    logits[3] = float("nan")
    for x, mask in ((logits, torch.zeros(100, dtype=torch.bool, device=DEV)), (logits[:0], None), (logits[:0], torch.zeros(0, dtype=torch.bool, device=DEV))):
        balance, z, counts, grad = _run(x, 2, mask, 1.0, 1.0)
        assert balance == 0.0 and z == 0.0 and not counts.view(torch.int32).any() and grad.shape == x.shape and not grad.any()


@pytest.mark.parametrize("dtype", _DTYPES)
def test_experts_that_are_switched_off(dtype):
    """-infinity and the type's lowest number: no probability, no gradient, chosen only where too few others are left"""
    T, E, k = 200, 20, 4
    logits = _logits(T, E, _DTYPES[dtype])
    open_ = logits[:, : E // 2].contiguous()
    want = _run(open_, k, None, 0.0, 1.0)
    for low in (-float("inf"), torch.finfo(logits.dtype).min):
        logits[:, E // 2 :] = low
        balance, z, counts, grad = _run(logits, k, None, 0.0, 1.0)
        assert torch.equal(counts.view(torch.int32)[: E // 2], want[2].view(torch.int32)) and not counts.view(torch.int32)[E // 2 :].any()
        assert not grad[:, E // 2 :].any() and torch.isfinite(grad).all()
        _check(open_, k, None, 0.0, 1.0, (want[0], z, want[2], grad[:, : E // 2].contiguous()))
        assert abs(float(balance) - 2.0 * float(want[0])) <= 2.0**-18 * float(balance)  # E is twice as large
    logits[:, 2:] = -float("inf")
    counts = fma.router_loss(logits, k)[2].view(torch.int32)
    assert counts.tolist() == [T] * k + [0] * (E - k)  # of the equal ones the first


@pytest.mark.parametrize("dtype", _DTYPES)
def test_logits_that_are_not_finite(dtype):
    """a token without a finite logit, with +infinity or NaN makes both losses NaN, as the formula has it; NaN is chosen before all numbers"""
    for bad in ("row", float("inf"), float("nan")):
        logits = _logits(50, 8, _DTYPES[dtype])
        if bad == "row":
            logits[7] = -float("inf")
        else:
            logits[7, 3] = bad
        balance, z, counts, grad = _run(logits, 2, None, 1.0, 1.0)
        assert torch.isnan(balance) and (torch.isnan(z) or (bad == float("inf") and torch.isinf(z)))
        assert torch.isnan(grad[7]).all() and int(counts.view(torch.int32).sum()) == 100
        if bad != "row":
            logits[7, 3] = 100.0
            assert torch.equal(fma.router_loss(logits, 2)[2].view(torch.int32), counts.view(torch.int32))


def test_large_logits():
    """magnitudes at which exp alone would overflow"""
    logits = _logits(500, 32, torch.float32, spread=1000.0)
    _check(logits, 4, None, 1.0, 1e-3)


def test_shapes_strides_and_offsets():
    base = _logits(6 * 40, 33, torch.bfloat16)
    _check(base.view(6, 40, 33), 3)
    mask = torch.rand(6, 40, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.5
    _check(base.view(6, 40, 33), 3, mask)
    _check(base, 3, mask)
    flat = _run(base, 3, mask, 1.0, 1.0)
    for other in (base.t().contiguous().t(), torch.cat([base, base], 1)[:, :33]):
        got = _run(other, 3, mask.t().contiguous().t(), 1.0, 1.0)
        assert got[0] == flat[0] and got[1] == flat[1] and torch.equal(got[3], flat[3])
    odd = _logits(1, 64 * 100 + 3, torch.float16)[0]
    for offset in (1, 2, 3):  # rows of whole vectors that start off a 16-byte boundary
        _check(odd[offset : offset + 6400].view(100, 64), 8)
    _check(_logits(1, 16, torch.float32)[0], 2)


def test_only_one_loss_is_used():
    logits = _logits(300, 16, torch.float32)
    for use, (gb, gz) in ((0, (1.0, 0.0)), (1, (0.0, 1.0))):
        leaf = logits.detach().requires_grad_()
        out = fma.router_loss(leaf, 2)
        out[use].backward()
        _check(logits, 2, None, gb, gz, (out[0].detach(), out[1].detach(), out[2], leaf.grad))
    assert not out[2].requires_grad
    with pytest.raises(RuntimeError):  # no second derivatives
        leaf = logits.detach().requires_grad_()
        (grad,) = torch.autograd.grad(fma.router_loss(leaf, 2)[1], leaf, create_graph=True)
        grad.sum().backward()


def test_gradient_against_differences():
    """central differences of the losses in 64 bits, the choice held fixed (the steps are far smaller than the gaps between the logits)"""
    T, E, k = 12, 8, 2
    logits = _logits(T, E, torch.float32)
    balance, z, counts, grad = _run(logits, k, None, 1.0, 0.5)
    f = counts.view(torch.int32).double() / (T * k)

    def loss(l64):
        return E * (f * torch.softmax(l64, -1).mean(0)).sum() + 0.5 * torch.logsumexp(l64, -1).square().mean()

    step = 1e-4
    for t in range(T):
        for e in range(E):
            d = torch.zeros(T, E, dtype=torch.float64, device=DEV)
            d[t, e] = step
            difference = (loss(logits.double() + d) - loss(logits.double() - d)) / (2 * step)
            # third derivatives are of the order of the gradients' own terms: step^2 of them
            assert abs(float(difference) - float(grad[t, e])) <= 1e-6 * float(grad.abs().max()) + 1e-10


def test_replays_from_a_captured_graph():
    static = _logits(700, 64, torch.bfloat16).requires_grad_()
    mask = torch.ones(700, dtype=torch.bool, device=DEV)
    grads = [torch.ones((), device=DEV), torch.full((), 0.5, device=DEV)]

    def step(leaf):
        leaf.grad = None
        balance, z, counts = fma.router_loss(leaf, 8, mask)
        torch.autograd.backward([balance, z], grads)
        return balance.detach(), z.detach(), counts, leaf.grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    static.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(static)
    for seed in range(1, 5):
        with torch.no_grad():
            static.copy_(_logits(700, 64, torch.bfloat16, seed))
        mask.copy_(torch.arange(700, device=DEV) % (seed + 1) > 0)
        graph.replay()
        torch.cuda.synchronize()
        want = step(static.detach().clone().requires_grad_())  # eager, between the replays
        torch.cuda.synchronize()
        assert held[0] == want[0] and held[1] == want[1] and torch.equal(held[3], want[3])
        assert torch.equal(held[2].view(torch.int32), want[2].view(torch.int32))


def test_two_streams_at_once():
    inputs = [_logits(30000, 64, torch.bfloat16, i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _run(inputs[i], 8, None, 1.0, 1.0)
    torch.cuda.synchronize()
    for x, g in zip(inputs, got):
        _check(x, 8, None, 1.0, 1.0, g)


def test_compiled_matches_eager():
    def f(logits, mask):
        balance, z, counts = fma.router_loss(logits, 4, mask)
        return balance, z, counts

    logits = _logits(333, 40, torch.bfloat16)
    mask = torch.arange(333, device=DEV) % 5 > 0
    out = []
    for fn in (f, torch.compile(f, fullgraph=True)):
        leaf = logits.detach().requires_grad_()
        balance, z, counts = fn(leaf, mask)
        (0.5 * balance + 0.25 * z).backward()
        out.append((balance.detach(), z.detach(), counts.view(torch.int32), leaf.grad))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_long_tensors():
    """logits past 2^31: the counts of the whole are those of its parts, the last tokens' gradients theirs alone"""
    E, k = 256, 8
    T = 2**31 // E + 5000
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device=DEV)
    logits[:, 0] = 1.0
    logits[-3000:] = _logits(3000, E, torch.bfloat16)
    mask = torch.zeros(T, dtype=torch.bool, device=DEV)
    mask[-3000:] = True
    _check(logits[-3000:], k, None, 0.7, -0.3, tuple(v if i < 3 else v[-3000:] for i, v in enumerate(_run(logits, k, mask, 0.7, -0.3))))
    counts = fma.router_loss(logits, k)[2].view(torch.int32).long()
    assert torch.equal(counts, sum(fma.router_loss(part, k)[2].view(torch.int32).long() for part in logits.split(T // 3)))


def test_a_second_pass_through_the_same_node():
    leaf = _logits(300, 40, torch.bfloat16).requires_grad_()
    balance, z, _ = fma.router_loss(leaf, 3)
    (balance + z).backward(retain_graph=True)
    first, leaf.grad = leaf.grad, None
    (balance + z).backward()
    assert torch.equal(first, leaf.grad)
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError):  # changed since, or freed by now
        (balance + z).backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_losses_of_the_layers_logits(dtype):
    """the counts are those of the experts that the layer ran, and the losses' gradients reach the gate and the tokens"""
    torch.manual_seed(3)
    moe = MoE(16, 4, 64, 32, swiglu_packed, True, False, 0.3).to(dtype).to(DEV)
    x = torch.randn(3, 50, 64, device=DEV).to(dtype).requires_grad_()
    y, logits = moe(x)
    mask = torch.arange(50, device=DEV).expand(3, 50) < torch.tensor([[50], [20], [0]], device=DEV)
    balance, z, counts = moe.router_loss(logits, mask)
    _check(logits.detach(), 4, mask, 0.7, -0.3, (balance.detach(), z.detach(), counts, _run(logits, 4, mask, 0.7, -0.3)[3]))
    if dtype == torch.bfloat16:  # (the fused router breaks ties the same way)
        selected = moe._compute_routing_weights(x.detach().view(-1, 64))[2].view(3, 50, 4)
        assert torch.equal(torch.bincount(selected[mask].reshape(-1), minlength=16), counts.view(torch.int32).long())
    (y.float().square().mean() + 0.01 * balance + 0.001 * z).backward()
    assert moe.gate.weight.grad.abs().max() > 0 and torch.isfinite(moe.gate.weight.grad).all() and torch.isfinite(x.grad).all()


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("E", [5, 8, 11, 32, 33, 64, 100, 160, 256, 300, 512, 700, 1024])
def test_every_small_number_of_choices(E, dtype):
    """1 to 17 choices: those around every power of two, of different logits, of few values, and of rows with as good as nothing but -infinity"""
    distinct = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i)) for i in range(65)]).to(DEV)
    distinct = ((distinct - E // 2).float() / 64).to(_DTYPES[dtype])  # (exact in every type up to 1024 experts: eleven bits, or rounded to equal ones)
    few = _logits(65, E, torch.float32).round().to(_DTYPES[dtype])
    rare = distinct.clone()
    rare[:, 3:] = -float("inf")
    for k in range(1, min(E, 17) + 1):
        for logits in (distinct, few):
            _check(logits, k)
        counts = fma.router_loss(rare, k)[2].view(torch.int32).long()
        chosen = torch.sort(rare.double(), dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(counts, torch.bincount(chosen.reshape(-1), minlength=E))


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("E", [8, 60, 256, 1024])
def test_choices_beside_a_nan(E, dtype):
    """a wavefront with one token that holds a NaN: the NaN comes first, and the other tokens choose as they do without it"""
    logits = _logits(200, E, _DTYPES[dtype])
    logits[77, E - 1] = float("nan")
    for k in (1, 2, 3, 8):
        order = logits.double()
        order[77, E - 1] = 1e9
        chosen = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(fma.router_loss(logits, k)[2].view(torch.int32).long(), torch.bincount(chosen.reshape(-1), minlength=E))
