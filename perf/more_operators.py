"""The operators of a training step around the MoE layer as cases that can be timed: the router's losses, the norm behind a block fused with its
gate, its residual scale and the norm before the next block, and the global norm of the gradients with their clipping.

A case is a dict of plain values. "op" says which entry point it runs:

  loss  router_loss, forward and backward: balance loss, z loss, tokens per expert, gradient of the logits
  norm  fused_sandwich_rmsnorm: both outputs, and with "train" the gradients of all inputs
  clip  clip_grad_norm_ on the gradients of a few layers: the norm and the clipped gradients

`own` False computes the same in elementary operations in 32 bits.
"""

import math
import os
import sys

import torch

own = False

if os.path.join(os.getcwd(), "cute-kernels_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "cute-kernels_amd"))  # the package's folder, from the repository's root

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5

# layer shapes of this repository's benchmark, tests and measurements: (H, I, E)
LAYERS = [(64, 128, 8), (256, 512, 8), (512, 344, 16), (512, 1024, 8), (2880, 2880, 32), (2048, 1024, 64), (2048, 1408, 64), (4096, 14336, 8)]


def _loss(T, E, k, dtype="bf16", padded=0.0):
    return dict(op="loss", T=T, E=E, k=k, dtype=dtype, padded=padded)


def _norm(N, S, H, dtype="bf16", gate="none", train=True, multiplier=1.0):
    return dict(op="norm", N=N, S=S, H=H, dtype=dtype, gate=gate, train=train, multiplier=multiplier)


def _clip(layers, shape, dtype="bf16", norm_type=2.0):
    H, I, E = shape
    return dict(op="clip", layers=layers, H=H, I=I, E=E, dtype=dtype, norm_type=norm_type)


def listed():
    return [
        # a small step in fp32, where launches count
        dict(_loss(512, 16, 2, "fp32"), name="loss_small_fp32"),
        # a batch of odd length with a third of it padding, fp16 and its loss scale
        dict(_loss(8191, 64, 8, "fp16", 0.3), name="loss_padded_fp16"),
        # the router of a training step over many experts
        dict(_loss(32768, 128, 8), name="loss_train"),
        # a large step in fp32
        dict(_loss(131072, 256, 8, "fp32"), name="loss_large_fp32"),
        # one user, one token, between two blocks
        dict(_norm(1, 1, 4096, train=False), name="norm_decode"),
        # a prefill chunk whose blocks have a scale per channel
        dict(_norm(1, 1021, 2048, "fp16", "channel", False), name="norm_prefill_fp16"),
        # a small step in fp32 with rows of odd length, the gate one row per sequence
        dict(_norm(4, 255, 1001, "fp32", "sequence", multiplier=0.5), name="norm_small_fp32"),
        # a training step with a gate for every element
        dict(_norm(4, 2047, 2880, gate="full", multiplier=0.22), name="norm_gated"),
        # the block around the large layer, no gate
        dict(_norm(4, 4096, 4096), name="norm_train"),
        # many small tensors: 24 layers
        dict(_clip(24, (64, 128, 8), "fp32"), name="clip_small_fp32"),
        # two layers of many experts
        dict(_clip(2, (2048, 1408, 64)), name="clip_experts"),
        # one layer of large experts
        dict(_clip(1, (4096, 14336, 8)), name="clip_large"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["loss", "norm", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "loss":
        E = rng.choice([4, 8, 16, 32, 33, 60, 64, 72, 128, 256, 1024])
        return _loss(_log_int(rng, 1, 131072 * 256 // max(E, 256)), E, rng.randint(1, min(E, 8)), dtype, rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "norm":
        H = rng.choice([64, 256, 512, 720, 1000, 1031, 1024, 2048, 2880, 4096, 8192])
        N = rng.choice([1, 2, 3, 8])
        S = _log_int(rng, 1, max(2, min(32768, 16384 * 4096 // 2 // H) // N))
        gate = rng.choice(["none", "none", "channel", "row", "sequence", "full"])
        return _norm(N, S, H, dtype, gate, rng.random() < 0.75, rng.choice([1.0, 0.22]))
    shape = rng.choice(LAYERS[:-1])
    H, I, E = shape
    layers = _log_int(rng, 1, min(24, max(1, 600_000_000 // (3 * H * I * E))))
    return _clip(layers, shape, dtype, rng.choice([2.0, 2.0, 2.0, math.inf]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, *shape):
    """N(0, 1) with a few wide channels, as hidden states have them"""
    return _randn(g, *shape) * torch.exp(0.5 * _randn(g, shape[-1]))


def _gate_shape(case):
    N, S, H = (case[n] for n in ("N", "S", "H"))
    return {"channel": (H,), "row": (N, S, 1), "sequence": (N, 1, H), "full": (N, S, H)}[case["gate"]]


def _layer_shapes(case):
    """the parameters of one block: two norms, the router, both projections of the experts"""
    H, I, E = (case[n] for n in ("H", "I", "E"))
    return [(H,), (H,), (E, H), (E, 2 * I, H), (E, H, I)]


def _elements(case):
    return case["layers"] * sum(math.prod(shape) for shape in _layer_shapes(case))


def prepare(case, seed):
    g = _generator(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "loss":
        T, E = case["T"], case["E"]
        logits = (_randn(g, T, E) + 0.5 * _randn(g, E)).to(dtype)  # some experts are preferred
        mask = torch.rand(T, generator=g, device="cuda") >= case["padded"] if case["padded"] else None
        # the losses' coefficients, times a loss scale where fp16 would lose the gradients otherwise
        scale = 2.0**16 if dtype is torch.float16 else 1.0
        grads = [torch.tensor(c * scale, device="cuda") for c in (0.01, 0.001)]
        return dict(op=op, logits=logits, mask=mask, k=case["k"], grads=grads)
    if op == "norm":
        N, S, H = (case[n] for n in ("N", "S", "H"))
        state = dict(op=op, train=case["train"], multiplier=case["multiplier"], gate=None)
        state["x"], state["residual"] = (_activations(g, N, S, H).to(dtype) for _ in range(2))
        state["post_weight"], state["weight"] = ((1.0 + 0.2 * _randn(g, H)).to(dtype) for _ in range(2))
        if case["gate"] != "none":
            state["gate"] = (0.5 + 0.3 * _randn(g, *_gate_shape(case))).to(dtype)
        if case["train"]:
            state["grads"] = [_randn(g, N, S, H).to(dtype) for _ in range(2)]
        return state
    # the gradients lie in one bucket, as a data-parallel program keeps them
    shapes = _layer_shapes(case) * case["layers"]
    bucket = (1e-3 * _randn(g, _elements(case))).to(dtype)
    bucket[::4096] *= 8.0  # a few large ones
    parameters = [torch.nn.Parameter(torch.empty(shape, dtype=dtype, device="cuda")) for shape in shapes]
    for p, grad in zip(parameters, bucket.split([math.prod(shape) for shape in shapes])):
        p.grad = grad.view(p.shape)
    norm = 1e-3 * math.sqrt(bucket.numel()) if case["norm_type"] == 2.0 else 4e-3
    return dict(op=op, parameters=parameters, bucket=bucket, max_norm=0.5 * norm, norm_type=case["norm_type"])


def _next_bound(s):
    """The bound of this pass. Passes over the same state clip what the last one has clipped; a bound that falls a little each time keeps
    every one of them a pass that has something to clip."""
    bound = s["max_norm"]
    s["max_norm"] = 0.999 * bound
    return bound


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _plain_loss(s):
    l32, k = s["logits"].float(), s["k"]
    T, E = l32.shape
    m = torch.ones(T, device="cuda") if s["mask"] is None else s["mask"].float()
    n = m.sum()
    p = torch.softmax(l32, -1)
    lse = torch.logsumexp(l32, -1)
    chosen = torch.sort(l32, dim=-1, descending=True, stable=True).indices[:, :k]
    counts = torch.zeros(E, device="cuda").index_add_(0, chosen.reshape(-1), m.repeat_interleave(k))
    one_over_n = torch.where(n > 0, 1.0 / n, 0.0)
    f = counts * one_over_n / k
    balance = E * (f * (m @ p) * one_over_n).sum()
    z = (m * lse.square()).sum() * one_over_n
    balance_grad, z_grad = s["grads"]
    grad = balance_grad * E * p * (f - (p * f).sum(-1, keepdim=True)) + 2.0 * z_grad * lse[:, None] * p
    grad = grad * (m * one_over_n)[:, None]
    return dict(balance=balance, z=z, counts=counts.to(torch.int32), logits_grad=grad.to(s["logits"].dtype))


def _unit(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_norm(s):
    names = [n for n in ("x", "residual", "post_weight", "weight", "gate") if s[n] is not None]
    t = {n: s[n].float().requires_grad_(s["train"]) for n in names}
    branch = _unit(t["x"]) * t["post_weight"]
    if "gate" in t:
        branch = branch * t["gate"]
    stream = t["residual"] + s["multiplier"] * branch
    normed = _unit(stream) * t["weight"]
    dtype = s["x"].dtype
    outputs = dict(normed=normed.detach().to(dtype), stream=stream.detach().to(dtype))
    if s["train"]:
        torch.autograd.backward([normed, stream], [grad.float() for grad in s["grads"]])
        outputs.update({n + "_grad": t[n].grad.to(dtype) for n in names})
    return outputs


def _plain_clip(s):
    bound, grads = _next_bound(s), [p.grad for p in s["parameters"]]
    if s["norm_type"] == 2.0:
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    else:
        norm = torch.stack([g.abs().max() for g in grads]).max().float()
    # (a factor of one dimension: one without any would be rounded to the gradients' type before the product)
    s["bucket"].mul_(torch.clamp(bound / (norm + 1e-6), max=1.0).view(1))
    return dict(norm=norm, grads=s["bucket"])


# ---- the framework's calls ------------------------------------------------------------------------------------------


def _leaf(t):
    return None if t is None else t.detach().requires_grad_()


def _own(s):
    import fma

    if s["op"] == "loss":
        logits = _leaf(s["logits"])
        balance, z, counts = fma.router_loss(logits, s["k"], s["mask"])
        torch.autograd.backward([balance, z], s["grads"])
        return dict(balance=balance.detach(), z=z.detach(), counts=counts.view(torch.int32), logits_grad=logits.grad)
    if s["op"] == "norm":
        names = ("x", "residual", "post_weight", "weight", "gate")
        if not s["train"]:
            with torch.no_grad():
                normed, stream = fma.fused_sandwich_rmsnorm(*(s[n] for n in names[:4]), EPS, s["gate"], s["multiplier"])
            return dict(normed=normed, stream=stream)
        # in float32 the leaves are the state's tensors, as in the plain form: gradients add up over passes, as in a program that accumulates them
        t = {n: s[n].requires_grad_() if s["x"].dtype is torch.float32 and s[n] is not None else _leaf(s[n]) for n in names}
        normed, stream = fma.fused_sandwich_rmsnorm(*(t[n] for n in names[:4]), EPS, t["gate"], s["multiplier"])
        torch.autograd.backward([normed, stream], s["grads"])
        grads = {n + "_grad": t[n].grad for n in names if t[n] is not None}
        return dict(normed=normed.detach(), stream=stream.detach(), **grads)
    norm = fma.clip_grad_norm_(s["parameters"], _next_bound(s), s["norm_type"])
    return dict(norm=norm, grads=s["bucket"])


_PLAIN = {"loss": _plain_loss, "norm": _plain_norm, "clip": _plain_clip}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def work(case):
    """bytes and operations of one pass: inputs read once, outputs written once"""
    op, s = case["op"], BYTES[case["dtype"]]
    if op == "loss":
        n = case["T"] * case["E"]
        return dict(bytes=2 * n * s, flops=20 * n)  # logits in, their gradient out
    if op == "norm":
        n = case["N"] * case["S"] * case["H"]
        gate = 0 if case["gate"] == "none" else math.prod(_gate_shape(case))
        if not case["train"]:
            return dict(bytes=(4 * n + gate) * s, flops=10 * n)  # x and residual in, both outputs out
        return dict(bytes=(8 * n + 2 * gate) * s, flops=40 * n)  # and both outputs' gradients in, those of x and residual out
    n = _elements(case)
    return dict(bytes=2 * n * s, flops=3 * n)


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------


def _exact_loss(s):
    logits, k = s["logits"].double(), s["k"]
    if s["mask"] is not None:
        kept = s["mask"].nonzero().flatten()
        logits = logits[kept]
    n, E = logits.shape
    total = torch.exp(logits).sum(1, keepdim=True)
    p, lse = torch.exp(logits) / total, torch.log(total)
    # an expert's place among a token's: how many logits are larger, or as large and further left
    place = torch.zeros_like(logits, dtype=torch.int32)
    for e in range(E):
        place += logits[:, e : e + 1] > logits
        place[:, e + 1 :] += logits[:, e : e + 1] == logits[:, e + 1 :]
    f = (place < k).double().sum(0) / max(1, n * k)
    balance = E * torch.dot(f, p.sum(0) / max(1, n))
    z = (lse * lse).sum() / max(1, n)
    balance_grad, z_grad = (grad.double() for grad in s["grads"])
    rows = (balance_grad * E * (f - (p @ f)[:, None]) + 2.0 * z_grad * lse) * p / max(1, n)
    if s["mask"] is not None:
        rows = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda").index_copy_(0, kept, rows)
    return dict(balance=balance, z=z, counts=None, logits_grad=rows)


def _exact_norm(s):
    x, residual, wp, w = (s[n].double() for n in ("x", "residual", "post_weight", "weight"))
    gate = torch.ones((), dtype=torch.float64, device="cuda") if s["gate"] is None else s["gate"].double()
    H, a = x.shape[-1], s["multiplier"]
    x_rms = torch.sqrt((x * x).sum(-1, keepdim=True) / H + EPS)
    stream = residual + a * gate * wp * x / x_rms
    rms = torch.sqrt((stream * stream).sum(-1, keepdim=True) / H + EPS)
    outputs = dict(normed=w * stream / rms, stream=stream)
    if not s["train"]:
        return outputs
    dy, dr = (grad.double() for grad in s["grads"])
    rows = tuple(range(x.dim() - 1))
    outputs["weight_grad"] = (dy * stream / rms).sum(rows)
    v = dy * w
    dr = dr + v / rms - stream * (v * stream).sum(-1, keepdim=True) / (H * rms**3)
    outputs["residual_grad"] = dr
    branch = a * dr * x / x_rms
    outputs["post_weight_grad"] = (branch * gate).sum(rows)
    if s["gate"] is not None:
        outputs["gate_grad"] = (branch * wp).sum_to_size(s["gate"].shape)
    v = a * dr * gate * wp
    outputs["x_grad"] = v / x_rms - x * (v * x).sum(-1, keepdim=True) / (H * x_rms**3)
    return outputs


def _exact_clip(s):
    grads = s["bucket"].double()
    norm = grads.pow(2).sum().sqrt() if s["norm_type"] == 2.0 else grads.abs().amax()
    return dict(norm=norm, grads=grads * min(1.0, s["max_norm"] / (float(norm) + 1e-6)))


def exact(case, seed):
    return {"loss": _exact_loss, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](prepare(case, seed))
