"""fused_sandwich_rmsnorm against its formulas in 64 bits, every output and gradient element by element.

Bounds, with u = 2^-24 and h half a step of the type. A mean over a row is off by n u of its terms' magnitudes, n = max(H / 256, 64) + 24 (a
thread adds at most that many one after the other, then threads and wavefronts join), an inverse root by half of that and three roundings.
Errors are carried through the formulas to first order, each product or sum adding one rounding of its terms; the backward pass starts from the
stream as it was before its rounding to the type. A sum over rows adds at most B / 256 + 40 roundings of its terms in 32 bits."""

import pytest
import torch

import fma

from gpu_util import DEV

pytestmark = pytest.mark.gpu

_U = 2.0**-24
_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}
_EPS = 1e-5
_NAMES = ("x", "residual", "post_weight", "weight", "gate")


def _gate_shape(kind, x_shape):
    N, S, H = x_shape
    return {"full": (N, S, H), "channel": (H,), "token": (N, S, 1), "sequence": (N, 1, H), "sequence_scalar": (N, 1, 1), "number": (1,)}[kind]


def _inputs(shape, dtype, gate="none", weights=True, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    H = shape[-1]
    t = dict(
        x=scale * randn(*shape), residual=randn(*shape), post_weight=1 + 0.3 * randn(H) if weights else None,
        weight=1 + 0.3 * randn(H) if weights else None, gate=None if gate == "none" else 0.5 + 0.5 * randn(*_gate_shape(gate, shape)),
    )  # fmt: skip
    return {n: None if v is None else v.to(dtype) for n, v in t.items()}, [randn(*shape).to(dtype) for _ in range(2)]


def _run(t, grads, a, eps=_EPS, function=fma.fused_sandwich_rmsnorm):
    leaves = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    out, stream = function(leaves["x"], leaves["residual"], leaves["post_weight"], leaves["weight"], eps, leaves["gate"], a)
    used = [(o, d) for o, d in zip((out, stream), grads) if d is not None]
    torch.autograd.backward([o for o, _ in used], [d for _, d in used])
    got = dict(out=out.detach(), stream=stream.detach())
    got.update({"d_" + n: v.grad for n, v in leaves.items() if v is not None})
    return got


def _exact(t, grads, a, eps=_EPS):
    """name -> (value, bound), in 64 bits"""
    x, residual = t["x"].double(), t["residual"].double()
    H, B = x.shape[-1], x.numel() // x.shape[-1]
    one = torch.ones(H, dtype=torch.float64, device=DEV)
    wp, w = (one if t[n] is None else t[n].double() for n in ("post_weight", "weight"))
    gate = torch.ones((), dtype=torch.float64, device=DEV) if t["gate"] is None else t["gate"].double()
    dy, dr_in = (torch.zeros_like(x) if d is None else d.double() for d in grads)
    dtype = t["x"].dtype
    h, n, acc = torch.finfo(dtype).eps / 2, max(H / 256, 64) + 24, B / 256 + 40
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    rounded = lambda v, e: (v, (e * (1 + 2.0**-8) + h * v.abs() * (1 + 2.0**-8) + _TINY[dtype]))  # noqa: E731

    inv_x = torch.rsqrt(mean(x * x) + eps)
    rel_x = (n / 2 + 3) * _U
    xh, exh = x * inv_x, (x * inv_x).abs() * (rel_x + 2 * _U)
    z = a * gate * wp * xh
    r = residual + z
    er = z.abs() * (rel_x + 6 * _U) + _U * r.abs()
    inv_r = torch.rsqrt(mean(r * r) + eps)
    rel_r = mean(r.abs() * er) / (mean(r * r) + eps) + (n / 2 + 3) * _U
    out = r * inv_r * w
    want = dict(out=rounded(out, w.abs() * inv_r * (er + r.abs() * (rel_r + 4 * _U))), stream=rounded(r, er))

    # backward
    rh, erh = r * inv_r, inv_r * er + (r * inv_r).abs() * (rel_r + 2 * _U)
    g = dy * w
    m = mean(g * rh)
    em = mean(g.abs() * erh) + (n + 4) * _U * mean((g * rh).abs())
    dr = dr_in + inv_r * (g - rh * m)
    terms = dr_in.abs() + inv_r * (g.abs() + (rh * m).abs())
    edr = inv_r * (rh.abs() * em + m.abs() * erh) + (6 * _U + rel_r) * terms
    want["d_residual"] = rounded(dr, edr)
    dz, edz, dz_terms = a * dr, abs(a) * edr + _U * (a * dr).abs(), abs(a) * terms
    gw = gate * wp
    v, ev, v_terms = dz * gw, gw.abs() * edz + 3 * _U * gw.abs() * dz_terms, gw.abs() * dz_terms
    mx = mean(v * xh)
    emx = mean(ev * xh.abs() + v.abs() * exh) + (n + 8) * _U * mean(v_terms * xh.abs())
    dx = inv_x * (v - xh * mx)
    want["d_x"] = rounded(dx, inv_x * (ev + xh.abs() * emx + mx.abs() * exh + (6 * _U + rel_x) * (v_terms + (xh * mx).abs())))

    def summed(value, error, shape, in_row=False):
        extra = (acc + (n if in_row else 0)) * _U * value.abs()
        return rounded(value.sum_to_size(shape), (error + extra).sum_to_size(shape))

    s, es = dz * xh, edz * xh.abs() + dz.abs() * exh + 3 * _U * dz_terms * xh.abs()
    if t["weight"] is not None:
        want["d_weight"] = summed(dy * rh, dy.abs() * erh + _U * (dy * rh).abs(), (H,))
    if t["post_weight"] is not None:
        want["d_post_weight"] = summed(s * gate, es * gate.abs() + 2 * _U * (s * gate).abs(), (H,))
    if t["gate"] is not None:
        want["d_gate"] = summed(s * wp, es * wp.abs() + 2 * _U * (s * wp).abs(), t["gate"].shape, t["gate"].shape[-1:] != (H,))
    return want


def _compare(got, want):
    for name, (value, bound) in want.items():
        assert got[name].shape == value.shape, name
        off = (got[name].double() - value).abs()
        assert bool((off <= bound).all()), f"{name}: {float((off / bound).max()):.3g} of the bound"


def _check(shape, dtype, gate="none", weights=True, a=0.7, seed=0, use=(True, True), scale=1.0):
    t, grads = _inputs(shape, dtype, gate, weights, seed, scale)
    grads = [d if u else None for d, u in zip(grads, use)]
    got = _run(t, grads, a)
    assert all(v.dtype == dtype for v in got.values())
    _compare(got, _exact(t, grads, a))
    return got


_GATES = ["none", "full", "channel", "token", "sequence", "sequence_scalar", "number"]
# rows of every length: below a vector, whole vectors and not, one to many vectors per thread, longer than registers hold
_LENGTHS = [1, 2, 3, 8, 9, 23, 64, 72, 128, 500, 512, 513, 1000, 1024, 1031, 2048, 2052, 2880, 4096, 4104, 8192, 8200, 16384, 16392, 20000, 32768, 65536]


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("gate", _GATES)
@pytest.mark.parametrize("H", _LENGTHS)
def test_against_fp64(H, gate, dtype):
    _check((3, 7, H), _DTYPES[dtype], gate)


# more rows than workgroups, sequences of one row, more sequences than workgroups, one long sequence, a single row
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("gate", _GATES)
@pytest.mark.parametrize("shape", [(1, 1, 96), (1, 1, 4096), (1, 3001, 64), (5, 1023, 48), (3001, 1, 40), (1501, 2, 72), (700, 3, 1024), (2, 1100, 2048), (2, 600, 4096), (1, 1200, 1001), (2500, 2, 72), (600, 2, 17000)])
def test_many_rows(shape, gate, dtype):
    _check(shape, _DTYPES[dtype], gate)


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("H", [65, 256, 2880])
@pytest.mark.parametrize("use", [(True, False), (False, True)])
@pytest.mark.parametrize("weights", [True, False])
def test_parts_left_out(H, dtype, use, weights):
    for gate in ("none", "channel", "token"):
        _check((2, 50, H), _DTYPES[dtype], gate, weights, use=use)


def test_a_gate_without_dimensions():
    t, grads = _inputs((2, 30, 96), torch.float32)
    t["gate"] = torch.tensor(0.7, device=DEV)
    _compare(_run(t, grads, 1.0), _exact(t, grads, 1.0))


def test_the_same_tensor_twice():
    """the block's output is its stream, and one scale serves both norms: each use adds to the gradient"""
    t, grads = _inputs((2, 30, 256), torch.bfloat16)
    t["residual"], t["weight"] = t["x"], t["post_weight"]
    want = _exact(t, grads, 1.0)
    x, w = t["x"].detach().requires_grad_(), t["weight"].detach().requires_grad_()
    out, stream = fma.fused_sandwich_rmsnorm(x, x, w, w, _EPS)
    torch.autograd.backward([out, stream], [d.expand_as(out) for d in grads], retain_graph=True)
    first = x.grad.clone(), w.grad.clone()
    for (a, b), grad in zip((("d_x", "d_residual"), ("d_weight", "d_post_weight")), first):
        value, bound = want[a][0] + want[b][0], want[a][1] + want[b][1]
        assert bool(((grad.double() - value).abs() <= bound + 2.0**-8 * value.abs() * 1.01).all())  # (and the sum of the two rounded)
    x.grad = w.grad = None
    torch.autograd.backward([out, stream], grads)  # a second time through the same node
    assert torch.equal(x.grad, first[0]) and torch.equal(w.grad, first[1])


@pytest.mark.parametrize("H", [60, 2048, 20000])
def test_one_weight_only(H):
    for missing in ("post_weight", "weight"):
        t, grads = _inputs((2, 30, H), torch.bfloat16, "sequence")
        t[missing] = None
        _compare(_run(t, grads, 1.0), _exact(t, grads, 1.0))


def test_multiplier_and_eps():
    t, grads = _inputs((40, 1, 512), torch.float32, "none")
    for a in (0.0, -1.5, 3.0):
        _compare(_run(t, grads, a), _exact(t, grads, a))
    same = [_run(t, grads, *args) for args in ((None,), (1.0,))]
    assert all(torch.equal(same[0][n], same[1][n]) for n in same[0])
    same = [_run(t, grads, 1.0, eps) for eps in (None, torch.finfo(torch.float32).eps)]
    assert all(torch.equal(same[0][n], same[1][n]) for n in same[0])
    _compare(_run(t, grads, 1.0, 0.5), _exact(t, grads, 1.0, 0.5))


@pytest.mark.parametrize("dtype", _DTYPES)
def test_rows_of_zeros(dtype):
    """a block that returned nothing: the stream passes, the gradient of x is that of x / sqrt(eps)"""
    for H in (64, 1001, 4096):
        t, grads = _inputs((2, 9, H), _DTYPES[dtype], "sequence", seed=1)
        t["x"][0] = 0
        got = _run(t, grads, 1.0)
        assert torch.equal(got["stream"][0], t["residual"][0]) and all(torch.isfinite(v).all() for v in got.values())
        if dtype != "fp16":  # (there 1 / sqrt(eps) of the upstream gradient)
            _compare(got, _exact(t, grads, 1.0))


@pytest.mark.parametrize("H", [64, 1001, 4096])
def test_a_row_that_is_not_finite_stays_one_row(H):
    t, grads = _inputs((2, 40, H), torch.bfloat16, "token")
    clean = _run(t, grads, 1.0)
    for bad in (float("nan"), float("inf")):
        t["x"][1, 7, 3] = bad
        got = _run(t, grads, 1.0)
        keep = torch.ones(2, 40, dtype=torch.bool, device=DEV)
        keep[1, 7] = False
        for n in ("out", "stream", "d_x", "d_residual", "d_gate"):
            assert torch.equal(got[n][keep], clean[n][keep]), n
        assert torch.isnan(got["out"][1, 7]).any() and torch.isnan(got["d_weight"]).any()


@pytest.mark.parametrize("H", [256, 1001])
def test_strides_and_alignment(H):
    t, grads = _inputs((6, 20, H), torch.bfloat16, "full")
    want = _run(t, grads, 1.0)

    def odd(v):  # the same numbers one element off a 16-byte boundary
        held = torch.empty(v.numel() + 1, dtype=v.dtype, device=DEV)
        held[1:] = v.reshape(-1)
        return held[1:].view(v.shape)

    forms = (
        odd,
        lambda v: v.transpose(0, -1).contiguous().transpose(0, -1),
        lambda v: torch.cat([v, v], -1)[..., : v.shape[-1]],
    )
    exact = _exact(t, grads, 1.0)
    for form in forms:
        got = _run({n: form(v) for n, v in t.items()}, [form(d) for d in grads], 1.0)
        _compare(got, exact)
        if form is not odd:  # (copied to contiguous tensors: the same kernels)
            assert all(torch.equal(got[n], want[n]) for n in want)


def test_same_bits_on_every_run():
    t, grads = _inputs((4, 900, 1024), torch.bfloat16, "sequence")
    runs = [_run(t, grads, 1.0) for _ in range(3)]
    assert all(torch.equal(runs[0][n], r[n]) for r in runs[1:] for n in r)


def test_without_rows():
    for gate in _GATES:
        t, grads = _inputs((0, 5, 64), torch.float32, gate)
        got = _run(t, grads, 1.0)
        assert got["out"].shape == got["d_x"].shape == (0, 5, 64) and not got["d_weight"].any() and not got["d_post_weight"].any()
        if gate != "none":
            assert got["d_gate"].shape == t["gate"].shape and not got["d_gate"].any()


def test_no_grad_gives_the_same_and_only_the_asked_gradients_are_made():
    t, grads = _inputs((2, 30, 256), torch.bfloat16, "channel")
    want = _run(t, grads, 1.0)
    with torch.no_grad():
        out, stream = fma.fused_sandwich_rmsnorm(t["x"], t["residual"], t["post_weight"], t["weight"], _EPS, t["gate"], 1.0)
    assert torch.equal(out, want["out"]) and torch.equal(stream, want["stream"]) and not out.requires_grad
    for name in ("gate", "weight", "post_weight", "x"):
        leaf = t[name].detach().requires_grad_()
        args = {**t, name: leaf}
        out, stream = fma.fused_sandwich_rmsnorm(args["x"], args["residual"], args["post_weight"], args["weight"], _EPS, args["gate"], 1.0)
        torch.autograd.backward([out, stream], grads)
        assert torch.equal(leaf.grad, want["d_" + name])
    with pytest.raises(RuntimeError):  # no second derivatives
        leaf = t["x"].detach().requires_grad_()
        out, _ = fma.fused_sandwich_rmsnorm(leaf, t["residual"], None, None, _EPS)
        (grad,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        grad.sum().backward()
    # a residual that is changed in place afterwards is noticed; the stream is not needed again and may be
    leaf, residual = t["x"].detach().requires_grad_(), t["residual"].clone()
    out, stream = fma.fused_sandwich_rmsnorm(leaf, residual, t["post_weight"], t["weight"], _EPS, t["gate"], 1.0)
    (stream + 0).backward(grads[1], retain_graph=True)
    with torch.no_grad():
        stream.mul_(0)
    out.backward(grads[0])
    parts = [_run(t, g, 1.0)["d_x"] for g in ((grads[0], None), (None, grads[1]))]
    assert torch.equal(leaf.grad, parts[0] + parts[1])
    leaf = t["x"].detach().requires_grad_()
    out, stream = fma.fused_sandwich_rmsnorm(leaf, residual, None, None, _EPS)
    with torch.no_grad():
        residual.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_gradient_against_differences():
    """central differences of the formula in 64 bits, for every input"""
    t, grads = _inputs((2, 3, 8), torch.float32, "sequence")
    got = _run(t, grads, 0.7)
    wide = {n: v.double() for n, v in t.items()}
    dy, dr = (d.double() for d in grads)

    def value(v):
        unit = lambda s: s / torch.sqrt(s.square().mean(-1, keepdim=True) + _EPS)  # noqa: E731
        stream = v["residual"] + 0.7 * v["gate"] * unit(v["x"]) * v["post_weight"]
        return float((unit(stream) * v["weight"] * dy).sum() + (stream * dr).sum())

    step = 1e-5
    for n in _NAMES:
        for i in range(wide[n].numel()):
            ends = []
            for sign in (1, -1):
                moved = wide[n].clone()
                moved.view(-1)[i] += sign * step
                ends.append(value({**wide, n: moved}))
            # step^2 of the third derivative, which is of the order of 1 / x^3 in the smallest rows
            assert abs((ends[0] - ends[1]) / (2 * step) - float(got["d_" + n].view(-1)[i])) <= 2e-5 * max(1.0, float(got["d_" + n].abs().max())), n


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
def test_replays_from_a_captured_graph(gate):
    shape = (3, 200, 512)
    t, grads = _inputs(shape, torch.bfloat16, gate)
    static = {n: None if v is None else v.clone().requires_grad_() for n, v in t.items()}

    def step(leaves, grads):
        for v in leaves.values():
            if v is not None:
                v.grad = None
        out, stream = fma.fused_sandwich_rmsnorm(leaves["x"], leaves["residual"], leaves["post_weight"], leaves["weight"], _EPS, leaves["gate"], 0.5)
        torch.autograd.backward([out, stream], grads)
        return [out.detach(), stream.detach()] + [v.grad for v in leaves.values() if v is not None]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, grads)
    torch.cuda.current_stream().wait_stream(side)
    for v in static.values():
        if v is not None:
            v.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(static, grads)
    for seed in range(1, 5):
        fresh, fresh_grads = _inputs(shape, torch.bfloat16, gate, seed=seed)
        with torch.no_grad():
            for n, v in fresh.items():
                if v is not None:
                    static[n].copy_(v)
            for d, f in zip(grads, fresh_grads):
                d.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        want = step({n: None if v is None else v.clone().requires_grad_() for n, v in fresh.items()}, fresh_grads)  # eager, between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_two_streams_at_once():
    sets = [_inputs((2, 3000, 512), torch.bfloat16, "channel", seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _run(*sets[i], 0.7)
    torch.cuda.synchronize()
    for (t, grads), g in zip(sets, got):
        _compare(g, _exact(t, grads, 0.7))


def test_compiled_matches_eager():
    for gate in ("none", "sequence"):
        t, grads = _inputs((2, 40, 256), torch.bfloat16, gate)
        eager = _run(t, grads, 0.5)
        compiled = _run(t, grads, 0.5, function=torch.compile(fma.fused_sandwich_rmsnorm, fullgraph=True))
        assert all(torch.equal(eager[n], compiled[n]) for n in eager)
    with torch.no_grad():
        outputs = torch.compile(fma.fused_sandwich_rmsnorm, fullgraph=True)(t["x"], t["residual"], t["post_weight"], t["weight"], _EPS, t["gate"], 0.5)
    assert torch.equal(outputs[0], eager["out"]) and torch.equal(outputs[1], eager["stream"])


def test_transforms_are_not_passed_over():
    """forward mode and functorch, which have no rule for this operator, raise; also without grad mode"""
    t, _ = _inputs((2, 3, 64), torch.float32)
    call = lambda x: fma.fused_sandwich_rmsnorm(x, t["residual"], None, None, _EPS)[0]  # noqa: E731
    with torch.no_grad(), pytest.raises(RuntimeError):
        with torch.autograd.forward_ad.dual_level():
            call(torch.autograd.forward_ad.make_dual(t["x"], torch.ones_like(t["x"])))
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.grad(lambda x: call(x).sum())(t["x"])


def test_long_tensors():
    """offsets past 2^31 elements"""
    B, H = 2**31 // 8192 + 40, 8192
    x = torch.zeros(B, H, dtype=torch.bfloat16, device=DEV)
    residual = torch.zeros_like(x)
    rows = torch.tensor([0, 1, B - 38, B - 1], device=DEV)
    t, grads = _inputs((1, 4, H), torch.bfloat16)
    x[rows], residual[rows] = t["x"][0], t["residual"][0]
    dy, dr = torch.zeros_like(x), torch.zeros_like(x)
    dy[rows], dr[rows] = grads[0][0], grads[1][0]
    x.requires_grad_()
    weight = t["weight"].detach().requires_grad_()
    out, stream = fma.fused_sandwich_rmsnorm(x, residual, t["post_weight"], weight, _EPS)
    torch.autograd.backward([out, stream], [dy, dr])
    want = _exact(t, grads, 1.0)
    _compare(dict(out=out.detach()[rows][None], stream=stream.detach()[rows][None], d_x=x.grad[rows][None], d_weight=weight.grad),
             {n: want[n] for n in ("out", "stream", "d_x", "d_weight")})


@pytest.mark.parametrize("H", [64, 1001, 4096])
def test_rows_of_zeros_in_fp16(H):
    """1 / sqrt(eps) = 316 times the upstream gradient, whose largest values here are below 65504 / 316 = 207"""
    t, grads = _inputs((2, 9, H), torch.float16, "sequence", seed=1)
    t["x"][0] = 0
    want = _exact(t, grads, 1.0)
    assert all(float(value.abs().max()) < 6e4 for value, _ in want.values())
    _compare(_run(t, grads, 1.0), want)
