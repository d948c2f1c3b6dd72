"""clip_grad_norm_, get_total_norm and clip_grads_with_norm_ against the formulas in 64 bits.

Tolerances: squares are added in 64 bits, so a norm is off by the rounding to float32, 2^-24 relative, and n 2^-53 for the sum. The factor is
one number for all elements, off by 2^-24 (rounded) of that norm's; an element is rounded in float32 (2^-24) and to its type (half a step)."""

import math

import pytest
import torch

import fma

from gpu_util import DEV

pytestmark = pytest.mark.gpu

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}  # half of the smallest number


def _parameters(grads):
    parameters = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        parameters.append(p)
    return parameters


def _norm64(grads, norm_type):
    if norm_type == math.inf:
        return max((float(g.double().abs().max()) for g in grads if g.numel()), default=0.0)
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check_norm(norm, want):
    assert norm.dtype == torch.float32 and norm.shape == () and norm.device == DEV
    assert abs(float(norm) - want) <= (2.0**-24 + 2.0**-30) * want


def _check_scaled(grads, before, want_norm, max_norm):
    factor = min(1.0, max_norm / (want_norm + 1e-6))
    for g, b in zip(grads, before):
        want = b.double() * factor
        if factor == 1.0:
            assert torch.equal(g, b)
            continue
        bound = want.abs() * (torch.finfo(g.dtype).eps / 2 + 3 * 2.0**-24) * (1 + 2.0**-20) + _TINY[g.dtype]
        assert bool(((g.double() - want).abs() <= bound).all())


def _draw(shapes, dtype, seed=0, scale=1e-2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(scale * torch.randn(s, generator=g, device=DEV)).to(dtype) for s in shapes]


# one element, sizes around a vector and around a chunk of 16384 elements, empty ones, more tensors than one table holds
SHAPES = {
    "one": [(1,)],
    "odd": [(3,), (8,), (0, 5), (7, 9), (1023,), (5, 1, 3)],
    "chunks": [(16383,), (16384,), (16385,), (3 * 16384 + 5,), ()],
    "many": [(1 + 37 * i % 301,) for i in range(391)],
    "layer": [(512,), (512,), (16, 512), (16, 688, 512), (16, 512, 344)],
}


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("shapes", SHAPES)
def test_against_fp64(shapes, dtype, norm_type):
    grads = _draw(SHAPES[shapes], _DTYPES[dtype])
    before = [g.clone() for g in grads]
    want = _norm64(before, norm_type)
    _check_norm(fma.get_total_norm(grads, norm_type), want)
    for share in (2.0, 0.37, 1e-3):
        for g, b in zip(grads, before):
            g.copy_(b)
        versions = [g._version for g in grads]
        norm = fma.clip_grad_norm_(_parameters(grads), share * want, norm_type)
        _check_norm(norm, want)
        _check_scaled(grads, before, want, share * want)
        assert [g._version for g in grads] == [v + 1 for v in versions]
        for g, b in zip(grads, before):
            g.copy_(b)
        assert fma.clip_grads_with_norm_(_parameters(grads), share * want, norm) is None
        _check_scaled(grads, before, float(norm), share * want)


def test_types_may_differ_and_order_does_not_change_the_bits():
    grads = _draw([(700, 33), (1,), (70001,)], torch.bfloat16) + _draw([(129,), (5000,)], torch.float32, 1) + _draw([(77, 7)], torch.float16, 2)
    want = _norm64(grads, 2.0)
    norms = [fma.get_total_norm(grads) for _ in range(3)]
    _check_norm(norms[0], want)
    assert norms[0] == norms[1] == norms[2]
    before = [g.clone() for g in grads]
    fma.clip_grad_norm_(_parameters(grads), 0.5 * want)
    _check_scaled(grads, before, want, 0.5 * want)


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("offset", [1, 3, 7])
def test_views_of_a_bucket(dtype, offset):
    """gradients back to back in one bucket, none of them on a 16-byte boundary; what lies around them stays as it is"""
    sizes = [5, 16384 + 3, 1, 40000]
    (bucket,) = _draw([(offset + sum(sizes) + 9,)], _DTYPES[dtype])
    before = bucket.clone()
    grads = list(bucket[offset : offset + sum(sizes)].split(sizes))
    was = [g.clone() for g in grads]
    want = _norm64(was, 2.0)
    _check_norm(fma.clip_grad_norm_(_parameters(grads), 0.25 * want), want)
    _check_scaled(grads, was, want, 0.25 * want)
    assert torch.equal(bucket[:offset], before[:offset]) and torch.equal(bucket[offset + sum(sizes) :], before[offset + sum(sizes) :])


def test_layouts():
    (base,) = _draw([(40, 30, 20)], torch.float32)
    before = base.clone()
    grads = [base[:10].permute(2, 0, 1), base[10:20, ::2], base[10:20, 1::2], base[20:30, :, 3:11], base[30:].transpose(0, 2)]
    was = [g.clone() for g in grads]
    parameters = [torch.nn.Parameter(torch.empty_like(g)) for g in was]
    for p, g in zip(parameters, grads):
        p.grad = g
    grads = [p.grad for p in parameters]
    want = _norm64(was, 2.0)
    _check_norm(fma.clip_grad_norm_(parameters, 0.5 * want), want)
    _check_scaled(grads, was, want, 0.5 * want)
    assert torch.equal(base[20:30, :, :3], before[20:30, :, :3]) and torch.equal(base[20:30, :, 11:], before[20:30, :, 11:])


def test_extreme_magnitudes():
    """squares beyond float32's range at both ends, subnormal elements, a norm that float32 does not hold"""
    for value, n, dtype in ((2.0**100, 1000, torch.bfloat16), (2.0**-100, 1000, torch.bfloat16), (2.0**-140, 77, torch.float32), (6e-8, 33, torch.float16), (65504.0, 4096, torch.float16)):
        g = torch.full((n,), value, device=DEV).to(dtype)
        want = float(g[0].double()) * math.sqrt(n)
        # (a result below float32's normal numbers is off by half of its smallest number)
        assert abs(float(fma.get_total_norm([g])) - want) <= 2.0**-23 * want + 2.0**-150
    g = torch.full((1 << 20,), 2.0**125, device=DEV).bfloat16()  # norm 2^135
    norm = fma.clip_grad_norm_(_parameters([g]), 1.0)
    assert float(norm) == math.inf and torch.equal(g, torch.full_like(g, 2.0**-10))


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_not_finite(bad, norm_type):
    grads = _draw([(100,), (20000,)], torch.bfloat16)
    grads[1][17777] = bad
    before = [g.clone() for g in grads]
    with pytest.raises(RuntimeError, match="finite"):
        fma.get_total_norm(grads, norm_type, error_if_nonfinite=True)
    with pytest.raises(RuntimeError, match="finite"):
        fma.clip_grad_norm_(_parameters(grads), 1.0, norm_type, error_if_nonfinite=True)
    assert all(torch.equal(g, b) or torch.isnan(b).any() for g, b in zip(grads, before)) and torch.equal(grads[0], before[0])
    norm = float(fma.clip_grad_norm_(_parameters(grads), 1.0, norm_type))
    # as the formula has it: a NaN norm makes everything NaN, an infinite one zero and the infinity itself NaN
    if math.isnan(bad):
        assert math.isnan(norm) and all(torch.isnan(g).all() for g in grads)
    else:
        assert norm == math.inf and not grads[0].any() and torch.isnan(grads[1]).sum() == 1


def test_zeros_and_a_bound_of_zero():
    grads = [torch.zeros(100, device=DEV), torch.zeros(0, device=DEV)]
    assert fma.clip_grad_norm_(_parameters(grads), 1.0) == 0.0 and not grads[0].any()
    grads = _draw([(100,)], torch.float32)
    fma.clip_grad_norm_(_parameters(grads), 0.0)
    assert not grads[0].any()
    assert fma.get_total_norm([torch.zeros(0, device=DEV)]) == 0.0


def test_parameters():
    (a, b) = _parameters(_draw([(300,), (20,)], torch.float32))
    unused = torch.nn.Parameter(torch.ones(4, device=DEV))
    want, was = _norm64([a.grad, b.grad], 2.0), [a.grad.clone(), b.grad.clone()]
    norm = fma.clip_grad_norm_((p for p in (a, unused, b, a)), 0.5 * want, error_if_nonfinite=True)  # a tied parameter counts once
    _check_norm(norm, want)
    _check_scaled([a.grad, b.grad], was, want, 0.5 * want)
    one = b.grad.clone()
    _check_norm(fma.clip_grad_norm_(b, math.inf), _norm64([one], 2.0))
    assert torch.equal(b.grad, one) and unused.grad is None
    _check_norm(fma.get_total_norm([one, one]), math.sqrt(2.0) * _norm64([one], 2.0))
    other = torch.nn.Parameter(torch.empty(20, device=DEV))
    other.grad = b.grad
    with pytest.raises(RuntimeError, match="share memory"):
        fma.clip_grad_norm_([b, other], 1e-3)
    other.grad = torch.ones(1, device=DEV).expand(20)
    with pytest.raises(RuntimeError, match="share memory"):
        fma.clip_grad_norm_([b, other], 1e-3)
    with pytest.raises(RuntimeError, match="one device"):
        fma.get_total_norm([one, one.cpu()])
    with pytest.raises(TypeError):
        fma.get_total_norm([one.double()])
    assert torch.equal(b.grad, one)


def test_gradients_that_a_graph_holds():
    """a gradient that autograd made with create_graph, and a backward that notices that it was changed"""
    x = torch.nn.Parameter(torch.full((50,), 2.0, device=DEV))
    (x**3).sum().backward(create_graph=True)
    want = _norm64([x.grad.detach()], 2.0)
    _check_norm(fma.clip_grad_norm_(x, 0.5 * want), want)
    assert x.grad.requires_grad
    y = torch.nn.Parameter(torch.ones(50, device=DEV))
    y.grad = torch.ones(50, device=DEV)
    loss = (y * y.grad).sum()
    fma.clip_grad_norm_(y, 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_replays_from_a_captured_graph():
    grads = _draw([(33,), (50000,), (128, 17)], torch.bfloat16)
    parameters = _parameters(grads)
    norm_static = None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fma.clip_grad_norm_(parameters, 0.5)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm_static = fma.clip_grad_norm_(parameters, 0.5)
    for seed in range(4):
        fresh = _draw([g.shape for g in grads], torch.bfloat16, seed, 10.0 ** (seed - 3))
        for g, f in zip(grads, fresh):
            g.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        want = fma.clip_grad_norm_(_parameters(fresh), 0.5)  # eager, between the replays
        torch.cuda.synchronize()
        assert norm_static == want and all(torch.equal(g, f) for g, f in zip(grads, fresh))


def test_two_streams_at_once():
    sets = [_draw([(100003,), (77,)], torch.float32, i) for i in range(2)]
    before = [[g.clone() for g in grads] for grads in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    norms = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for g, b in zip(sets[i], before[i]):
                    g.copy_(b)
                norms[i] = fma.clip_grad_norm_(_parameters(sets[i]), 0.5)
    torch.cuda.synchronize()
    for i in range(2):
        want = _norm64(before[i], 2.0)
        _check_norm(norms[i], want)
        _check_scaled(sets[i], before[i], want, 0.5)


def test_compiled_function_breaks_its_graph_here():
    grads = _draw([(100,), (2000,)], torch.float32)
    parameters, before = _parameters(grads), [g.clone() for g in grads]

    def step(scale):
        norm = fma.clip_grad_norm_(parameters, 0.5)
        return norm * scale

    want = _norm64(before, 2.0)
    got = torch.compile(step)(torch.ones((), device=DEV))
    _check_norm(got, want)
    _check_scaled(grads, before, want, 0.5)


def test_long_tensors():
    """elements past 2^31, and a set that is read and written as a stream"""
    n = 2**31 + 16384 + 5
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    places = torch.tensor([0, 1, 2**31 - 1, 2**31, 2**31 + 16383, n - 1], device=DEV)
    g[places] = torch.arange(1.0, 7.0, device=DEV).bfloat16()
    small = torch.full((3,), 2.0, device=DEV)
    norm = fma.clip_grad_norm_(_parameters([small, g]), 0.5)
    want = math.sqrt(91.0 + 12.0)
    _check_norm(norm, want)
    factor = 0.5 / (want + 1e-6)
    for got, exact in ((g[places].double(), torch.arange(1.0, 7.0, device=DEV).double() * factor), (small.double(), small.new_full((3,), 2.0).double() * factor)):
        assert bool(((got - exact).abs() <= exact * 2.0**-8 * 1.001).all())
    assert int(torch.count_nonzero(g)) == 6
    _check_norm(fma.get_total_norm([g], math.inf), float(g[n - 1].double()))


def test_strided_gradients_that_share_memory():
    """one view twice is refused; views that lie between each other are clipped as ever"""
    base = torch.randn(40, 30, device=DEV)
    same = _parameters([base[:, ::2], base[:, ::2]])
    before = base.clone()
    with pytest.raises(RuntimeError, match="share memory"):
        fma.clip_grad_norm_(same, 1e-3)
    with pytest.raises(RuntimeError, match="share memory"):
        fma.clip_grads_with_norm_(same, 1e-3, torch.tensor(1.0, device=DEV))
    assert torch.equal(base, before)
    norm = fma.clip_grad_norm_(_parameters([base[:, ::2], base[:, 1::2]]), 1e-3)
    _check_norm(norm, float(before.double().norm()))
    _check_scaled([base], [before], float(before.double().norm()), 1e-3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("magnitude,max_norm", [(2.0**125, 0.37), (2.0**125, 1e-6), (2.0**125, 1e-30), (2.0**125, 1.5e-37), (1e10, 1e-33), (1e-2, 1.5e-37)])
def test_factors_below_float32s_normal_numbers(magnitude, max_norm, dtype):
    """The factor lies where float32 has few bits or none, the results do not (or only just). The factor's leading digits are rounded once, as
    ever; scaling by a power of two rounds only a result that is itself below the normal numbers, by half of float32's smallest."""
    g = torch.Generator(device=DEV).manual_seed(5)
    before = (magnitude * (1.0 + 0.9 * torch.rand(1 << 20, generator=g, device=DEV)) * (1 - 2 * (torch.rand(1 << 20, generator=g, device=DEV) < 0.5))).to(dtype)
    norm = _norm64([before], 2.0)
    calls = [(norm, lambda p: fma.clip_grad_norm_(p, max_norm))]
    if norm < 2.0**127:
        given = torch.tensor(norm, device=DEV)
        calls.append((float(given.double()), lambda p: fma.clip_grads_with_norm_(p, max_norm, given)))
    for norm, call in calls:
        (p,) = _parameters([before.clone()])
        call([p])
        factor = max_norm / (norm + 1e-6)
        assert 0.0 < factor < 2.0**-126
        want = before.double() * factor
        bound = want.abs() * (torch.finfo(dtype).eps / 2 + 3 * 2.0**-24) * (1 + 2.0**-20) + _TINY[dtype] + 2.0**-150
        assert bool(((p.grad.double() - want).abs() <= bound).all()) and bool(p.grad.any())


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_a_total_norm_in_64_bits(where):
    """Scaling goes by its 64 bits: the factor is rounded to float32, the norm is not. Expected bits: factor and product in IEEE arithmetic."""
    (before,) = _draw([(5003,)], torch.float32)
    for i in range(24):
        norm, max_norm = 3.0 + 1e-8 * (i + 1) / 7, 0.1 + 0.013 * i
        (p,) = _parameters([before.clone()])
        fma.clip_grads_with_norm_([p], max_norm, torch.tensor(norm, dtype=torch.float64, device=where))
        factor = torch.tensor(max_norm / (norm + 1e-6), dtype=torch.float64).float().to(DEV)
        assert torch.equal(p.grad, before * factor)
    large = torch.full((77,), 1e30, device=DEV)
    (p,) = _parameters([large.clone()])
    fma.clip_grads_with_norm_([p], 1.0, torch.tensor(1e40, dtype=torch.float64, device=where))
    want = large.double() * (1.0 / (1e40 + 1e-6))
    assert bool(((p.grad.double() - want).abs() <= want * 3 * 2.0**-24).all())
    whole = torch.tensor(2**24 + 3, device=where)  # a whole number that float32 does not hold: there it is one more
    (p,) = _parameters([torch.ones(3, device=DEV)])
    fma.clip_grads_with_norm_([p], float(2**24 + 3) + 1e-6, whole)
    assert torch.equal(p.grad, torch.ones(3, device=DEV))


@pytest.mark.parametrize("dtype", _DTYPES)
def test_the_check_for_finite_norms_changes_no_bit(dtype):
    """error_if_nonfinite adds a look at the norm, and scales by the same one"""
    before = _draw([(1001, 37), (5,), (4099,)], _DTYPES[dtype])
    for i in range(1, 25):
        ends = []
        for check in (False, True):
            grads = [b.clone() for b in before]
            norm = fma.clip_grad_norm_(_parameters(grads), 0.01 * i, error_if_nonfinite=check)
            ends.append([norm] + grads)
        assert all(torch.equal(a, b) for a, b in zip(*ends))


def test_a_finite_norm_that_float32_does_not_hold_is_finite():
    before = torch.full((1 << 20,), 2.0**125, device=DEV).bfloat16()  # norm 2^135
    ends = []
    for check in (False, True):
        g = before.clone()
        assert float(fma.clip_grad_norm_(_parameters([g]), 3.0, error_if_nonfinite=check)) == math.inf
        ends.append(g)
    assert torch.equal(*ends) and torch.equal(ends[0], torch.full_like(before, 1.5 * 2.0**-9))
    with pytest.raises(RuntimeError, match="finite"):  # what is returned here is not
        fma.get_total_norm([before], error_if_nonfinite=True)


def test_tensors_in_another_order():
    """the norm is within its bound whatever the order, and each tensor is scaled by the same factor"""
    grads = _draw([(700, 33), (1,), (70001,)], torch.bfloat16) + _draw([(129,), (5000,)], torch.float32, 1) + _draw([(77, 7)], torch.float16, 2)
    want = _norm64(grads, 2.0)
    for order in ((5, 4, 3, 2, 1, 0), (2, 0, 5, 1, 4, 3), (3, 5, 0, 4, 2, 1)):
        some = [grads[i].clone() for i in order]
        before = [g.clone() for g in some]
        _check_norm(fma.get_total_norm(some), want)
        _check_norm(fma.clip_grad_norm_(_parameters(some), 0.5 * want), want)
        _check_scaled(some, before, want, 0.5 * want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nothing_is_written_where_the_norm_is_refused(bad):
    grads = _draw([(100,), (20000,)], torch.bfloat16)
    grads[1][17777] = bad
    before, versions = [g.clone() for g in grads], [g._version for g in grads]
    with pytest.raises(RuntimeError, match="finite"):
        fma.clip_grad_norm_(_parameters(grads), 1e-3, error_if_nonfinite=True)
    assert all(torch.equal(g.view(torch.int16), b.view(torch.int16)) for g, b in zip(grads, before))
    assert [g._version for g in grads] == versions


def test_a_dense_gradient_and_a_view_into_it():
    """views that differ and overlap: every element is scaled once, and counts as often as it is named in the norm"""
    base = torch.randn(40, 30, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    before = base.clone()
    norm = math.sqrt(float(before.double().square().sum()) + float(before[:, ::2].double().square().sum()))
    _check_norm(fma.clip_grad_norm_(_parameters([base, base[:, ::2]]), 0.5 * norm), norm)
    _check_scaled([base], [before], norm, 0.5 * norm)


def test_a_norm_that_is_an_element_of_a_gradient():
    """refused where the kernels would write it, and right where they write a copy of the gradient or where it only lies beside it"""
    (bucket,) = _draw([(5000,)], torch.float32)
    bucket[4000] = 2.0
    before = bucket.clone()
    (p,) = _parameters([bucket])
    with pytest.raises(RuntimeError, match="norm shares memory"):
        fma.clip_grads_with_norm_([p], 1.0, bucket[4000])
    assert torch.equal(bucket, before)
    (strided,) = _parameters([bucket[::2]])
    fma.clip_grads_with_norm_([strided], 1.0, bucket[4000])
    _check_scaled([strided.grad], [before[::2]], 2.0, 1.0)
    bucket.copy_(before)
    parts = _parameters([bucket[:4000], bucket[4001:]])
    fma.clip_grads_with_norm_(parts, 1.0, bucket[4000])
    _check_scaled([q.grad for q in parts], [before[:4000], before[4001:]], 2.0, 1.0)
    assert bucket[4000] == 2.0
