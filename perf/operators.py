"""The 8-bit operators as cases that can be timed: quantisation to blocks of 128, products of quantised operands, the SwiGLU activation
that keeps its input in 8 bits, and the expert path of the MoE layer made of them.

A case is a dict of plain values. "op" says which entry point it runs:

  quantize  quantize_fp8: one scale per 1 x 128 (block_rows 1) or 128 x 128 (block_rows 128, with the transposed copy) elements
  product   grouped_gemm_fp8 on operands that are in 8 bits already: a serving product
  linear    grouped_linear_fp8, forward and backward: output, gradients of the rows and of the weights
  swiglu    swiglu_packed_fp8, the activation that keeps its input in 8 bits, forward and backward
  infer     swiglu_experts_fp8 on weights that are in 8 bits already, no backward
  train     swiglu_experts_fp8 on 16-bit weights, forward and backward: output, gradients of tokens, router weights and both weights

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
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

# layer shapes of this repository's benchmark, tests and measurements: (H, I, E, k)
SHAPES = [
    (4096, 14336, 8, 2),
    (2048, 1408, 64, 8),
    (4096, 1536, 128, 8),
    (2048, 8192, 8, 2),
    (2048, 1024, 64, 8),
    (2880, 2880, 32, 4),
    (2048, 768, 128, 8),
]


def _layer(op, T, shape, dtype="bf16", skew=0.0):
    H, I, E, k = shape
    return dict(op=op, T=T, H=H, I=I, E=E, k=k, dtype=dtype, skew=skew)


def _rows(op, R, E, N, K, dtype="bf16", skew=0.0):
    return dict(op=op, R=R, E=E, N=N, K=K, dtype=dtype, skew=skew)


def listed():
    return [
        # the tokens of a training step on their way into the first product
        dict(op="quantize", E=1, N=16384, K=4096, block_rows=1, dtype="bf16", name="quantize_tokens"),
        # all experts' first projections at the start of a training step: the blocks, and the copy that the input gradient reads
        dict(op="quantize", E=64, N=2816, K=2048, block_rows=128, dtype="bf16", name="quantize_weights"),
        # a decode step's first projection: a few rows per expert against all weights
        dict(_rows("product", 32, 8, 28672, 4096), name="product_decode"),
        # a prompt of odd length, unevenly routed, a reduction that ends inside a block, fp16 out
        dict(_rows("product", 1021 * 4, 32, 5760, 2880, dtype="fp16", skew=0.5), name="product_ragged_fp16"),
        # the first projection of a large prefill on few large experts
        dict(_rows("product", 32768, 8, 28672, 4096), name="product_large_experts"),
        # one projection of a small step, where launches and host work count
        dict(_rows("linear", 509, 8, 1024, 512, dtype="fp16"), name="linear_small_fp16"),
        # one projection of a training step over many experts, some of them preferred
        dict(_rows("linear", 65536, 64, 2048, 1408, skew=0.5), name="linear_train"),
        # the activation of a training step: forward and backward
        dict(op="swiglu", R=65536, I=1408, dtype="bf16", name="swiglu_train"),
        # a small one of odd length in fp32
        dict(op="swiglu", R=509, I=344, dtype="fp32", name="swiglu_small_fp32"),
        # one user, one token: launches and their latencies count
        dict(_layer("infer", 1, (2048, 1408, 64, 8)), name="experts_decode_1"),
        # a prefill chunk over many experts
        dict(_layer("infer", 4096, (4096, 1536, 128, 8)), name="experts_prefill"),
        # the expert path of a training step
        dict(_layer("train", 8192, (2048, 1408, 64, 8), skew=0.25), name="experts_train"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choices(["quantize", "product", "linear", "swiglu", "infer", "train"], [3, 5, 3, 2, 4, 2])[0]
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16"])
    skew = rng.choice([0.0, 0.0, 0.25, 0.5])
    if op == "quantize":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        if rng.random() < 0.6:
            return dict(op=op, E=1, N=_log_int(rng, 1, 32768), K=rng.choice([768, 1408, 2048, 2880, 4096, 8192]), block_rows=1, dtype=dtype)
        H, I, E, _ = rng.choice(SHAPES[1:])
        return dict(op=op, E=max(1, E // rng.choice([1, 4, 8])), N=I, K=H, block_rows=128, dtype=dtype)
    if op == "swiglu":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return dict(op=op, R=_log_int(rng, 1, 65536), I=rng.choice([344, 768, 1024, 1408, 1536, 2880]), dtype=dtype)
    H, I, E, k = shape = rng.choice(SHAPES)
    if op in ("product", "linear"):
        N, K = rng.choice([(2 * I, H), (H, I), (H, 16 * rng.randint(8, 256))])
        most = 2.0 * 32768 * 28672 * 4096 if op == "product" else 2.0 * 65536 * 2048 * 1408
        rows = int(min(32768 if op == "product" else 65536, most / (2.0 * N * K)))
        return _rows(op, _log_int(rng, 1 if op == "product" else 64, rows), E, N, K, dtype, skew)
    largest = 2.0 * 32768 * 28672 * 4096
    if op == "infer":
        most = int(min(8192, largest / (6.0 * k * H * I)))
        return _layer(op, _log_int(rng, 1, most), shape, dtype, skew)
    most = int(min(8192, largest / (4 * 6.0 * k * H * I)))
    return _layer(op, _log_int(rng, 128, most), rng.choice([shape, SHAPES[1]]), dtype, skew)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, width):
    """N(0, 1) with a few wide channels, as hidden states have them"""
    x = _randn(g, rows, width)
    return x * torch.exp(0.5 * _randn(g, width))


def _logits(g, rows, E, skew):
    return _randn(g, rows, E) + 3.0 * skew * _randn(g, E)


def _group_sizes(g, R, E, skew):
    """uint32 [E]: rows of every group, R in all"""
    choice = torch.multinomial(torch.softmax(_logits(g, 1, E, skew)[0] * skew, 0), R, replacement=True, generator=g)
    return torch.bincount(choice, minlength=E).to(torch.int32).view(torch.uint32)


def prepare(case, seed):
    g = _generator(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    state = dict(op=op, dtype=dtype)
    if op == "quantize":
        x = _activations(g, case["E"] * case["N"], case["K"]) if case["block_rows"] == 1 else 0.02 * _randn(g, case["E"] * case["N"], case["K"])
        return dict(state, x=x.to(dtype).view(case["E"], case["N"], case["K"]), block_rows=case["block_rows"])
    if op == "swiglu":
        return dict(state, x=_activations(g, case["R"], 2 * case["I"]).to(dtype), dy=_randn(g, case["R"], case["I"]).to(dtype))
    if op in ("product", "linear"):
        R, E, N, K = (case[n] for n in ("R", "E", "N", "K"))
        sizes = _group_sizes(g, R, E, case["skew"])
        state.update(M_array=sizes, most=int(sizes.view(torch.int32).max()))
        x, w = _activations(g, R, K).to(dtype), (0.02 * _randn(g, E, N, K)).to(dtype)
        if op == "product":
            return dict(state, x=_quantize(x), w=_quantize(w, 128))
        return dict(state, x=x, w=w, dy=_randn(g, R, N).to(dtype))
    T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
    gates, selected = torch.topk(_logits(g, T, E, case["skew"]), k, dim=-1)
    sizes = torch.bincount(selected.reshape(-1), minlength=E)
    state.update(gates=torch.softmax(gates, -1).to(dtype), selected=selected.to(torch.int32), most=int(sizes.max()), E=E)
    x, w1, w2 = _activations(g, T, H).to(dtype), (0.02 * _randn(g, E, 2 * I, H)).to(dtype), (0.02 * _randn(g, E, H, I)).to(dtype)
    if op == "infer":  # (the up and the gate projection of an expert are quantised as two matrices)
        return dict(state, x=x, w1=_quantize(w1.view(E, 2, I, H), 128), w2=_quantize(w2, 128))
    return dict(state, x=x, w1=w1, w2=w2, dy=_randn(g, T, H).to(dtype))


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _blocks(x, block_rows):
    """x [.., N, K] as blocks [.., n, block_rows, k, 128], zeros past its ends"""
    N, K = x.shape[-2:]
    x = torch.nn.functional.pad(x.float(), (0, -K % 128, 0, -N % block_rows))
    return x.unflatten(-1, (-1, 128)).unflatten(-3, (-1, block_rows))


def _quantize(x, block_rows=1):
    """(values, scales): the smallest power of two that brings a block's largest magnitude to 448 or less, 2^-126 at the least, and the
    block divided by it; a block with an infinity or a NaN is NaN. Rows of scales are filled up with ones to a multiple of four."""
    blocks = _blocks(x, block_rows)
    amax = blocks.abs().amax((-3, -1), keepdim=True)
    fine = torch.isfinite(amax)
    # 448 = 1.75 * 2^8: the exponent of amax / 448, rounded up, in the bits of amax
    byte = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=1)
    inverse = ((254 - byte) << 23).view(torch.float32)
    values = torch.where(fine, blocks * inverse, math.nan).flatten(-4, -3).flatten(-2)[..., : x.shape[-2], : x.shape[-1]].to(E4M3)
    byte = torch.where(fine, byte, 255).to(torch.uint8).squeeze(-1).squeeze(-2)
    return values.contiguous(), torch.nn.functional.pad(byte, (0, -byte.shape[-1] % 4), value=127).view(E8M0).contiguous()


def _transpose_blocks(values, scales):
    """the transposed copy of a matrix quantised in 128 x 128 blocks"""
    n, k = scales.shape[-2], (values.shape[-1] + 127) // 128
    byte = scales.view(torch.uint8)[..., :k].transpose(-1, -2)
    values = values.view(torch.uint8).transpose(-1, -2).contiguous().view(E4M3)
    return values, torch.nn.functional.pad(byte, (0, -n % 4), value=127).view(E8M0).contiguous()


def _dequantize(blocks, block_rows=1):
    values, scales = blocks
    N, K = values.shape[-2:]
    byte = scales.view(torch.uint8).int()
    scale = torch.where(byte == 255, math.nan, (byte << 23).view(torch.float32))
    scale = scale.repeat_interleave(block_rows, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]
    return values.float() * scale


def _seen_in_8_bits(x, block_rows=1):
    return _dequantize(_quantize(x, block_rows), block_rows)


def _places(sizes, R):
    """expert and place within the expert of every row, where the rows of the experts lie back to back"""
    sizes = sizes.view(torch.int32).long()
    expert = torch.repeat_interleave(sizes, output_size=R)
    return expert, torch.arange(R, device="cuda") - (sizes.cumsum(0) - sizes)[expert]


def _spread(x, places, E, most):
    """rows back to back -> [E, most, width], zeros behind the rows of an expert"""
    out = x.new_zeros(E, most, x.shape[1])
    out[places] = x
    return out


def _grouped(x, w, places, most):
    """x_e w_e^T of every expert, rows back to back"""
    return torch.bmm(_spread(x, places, w.shape[0], most), w.transpose(1, 2).contiguous())[places]


def _grouped_weight_grad(dy, x, places, E, most):
    """dy_e^T x_e of every expert"""
    return torch.bmm(_spread(dy, places, E, most).transpose(1, 2).contiguous(), _spread(x, places, E, most))


def _swiglu(up, gate):
    return up * gate * torch.sigmoid(gate)


def _swiglu_grad(up, gate, dy):
    s = torch.sigmoid(gate)
    return torch.cat((dy * gate * s, dy * up * (s + gate * s * (1.0 - s))), -1)


def _halves_in_8_bits(h):
    """[up | gate] with each half quantised apart"""
    return _seen_in_8_bits(h.unflatten(-1, (2, -1))).flatten(-2)


def _plain_linear(s):
    dtype, x, w, dy = s["dtype"], s["x"], s["w"], s["dy"].float()
    places = _places(s["M_array"], x.shape[0])
    x, w = _seen_in_8_bits(x), _seen_in_8_bits(w, 128)
    y = _grouped(x, w, places, s["most"])
    x_grad = _grouped(_seen_in_8_bits(dy), w.transpose(1, 2), places, s["most"])
    w_grad = _grouped_weight_grad(dy, x, places, w.shape[0], s["most"])
    return dict(y=y.to(dtype), x_grad=x_grad.to(dtype), w_grad=w_grad.to(dtype))


def _plain_experts(s):
    dtype, E, most, gates = s["dtype"], s["E"], s["most"], s["gates"].float()
    T, k = gates.shape
    expert, slot = s["selected"].reshape(-1).long().sort(stable=True)
    sizes = torch.zeros(E, dtype=torch.long, device="cuda").index_add_(0, expert, torch.ones_like(expert))
    places = expert, torch.arange(T * k, device="cuda") - (sizes.cumsum(0) - sizes)[expert]
    token = slot // k
    training = s["op"] == "train"
    x = _seen_in_8_bits(s["x"])
    if training:
        w1 = _seen_in_8_bits(s["w1"].unflatten(1, (2, -1)), 128).flatten(1, 2)
        w2 = _seen_in_8_bits(s["w2"], 128)
    else:
        w1, w2 = _dequantize(s["w1"], 128).flatten(1, 2), _dequantize(s["w2"], 128)
    h = _grouped(x[token], w1, places, most)
    act = _seen_in_8_bits(_swiglu(*h.chunk(2, -1)))
    o = _grouped(act, w2, places, most)
    gate = gates.reshape(-1)[slot].unsqueeze(1)
    per_token = lambda rows: torch.empty_like(rows).index_copy_(0, slot, rows).view(T, k, -1).sum(1)  # noqa: E731
    y = per_token(o * gate)
    if not training:
        return y.to(dtype)
    dy = s["dy"].float()[token]
    gates_grad = torch.empty(T * k, device="cuda").index_copy_(0, slot, (dy * o).sum(-1)).view(T, k)
    o_grad = dy * gate
    h_grad = _swiglu_grad(*_halves_in_8_bits(h).chunk(2, -1), _grouped(_seen_in_8_bits(o_grad), w2.transpose(1, 2), places, most))
    grouped_grad = _grouped(_halves_in_8_bits(h_grad), w1.transpose(1, 2), places, most)
    x_grad = per_token(grouped_grad)
    w1_grad = _grouped_weight_grad(h_grad, x[token], places, E, most)
    w2_grad = _grouped_weight_grad(o_grad, act, places, E, most)
    return dict(y=y.to(dtype), x_grad=x_grad.to(dtype), gates_grad=gates_grad.to(dtype), w1_grad=w1_grad.to(dtype), w2_grad=w2_grad.to(dtype))


def _plain(s):
    op, dtype = s["op"], s["dtype"]
    if op == "quantize":
        blocks = _quantize(s["x"], s["block_rows"])
        return [*blocks] if s["block_rows"] == 1 else [*blocks, *_transpose_blocks(*blocks)]
    if op == "product":
        x = _dequantize(s["x"])
        return _grouped(x, _dequantize(s["w"], 128), _places(s["M_array"], x.shape[0]), s["most"]).to(dtype)
    if op == "linear":
        return _plain_linear(s)
    if op == "swiglu":
        x = s["x"].float()
        y = _swiglu(*x.chunk(2, -1))
        x_grad = _swiglu_grad(*_halves_in_8_bits(x).chunk(2, -1), s["dy"].float())
        return dict(y=y.to(dtype), x_grad=x_grad.to(dtype))
    return _plain_experts(s)


# ---- the framework's calls ------------------------------------------------------------------------------------------


def _leaf(t):
    return t.detach().requires_grad_()


def _own(s):
    import fma

    op = s["op"]
    if op == "quantize":
        if s["block_rows"] == 1:
            return [*fma.quantize_fp8(s["x"])]
        blocks, transposed = fma.quantize_fp8(s["x"], block_rows=128, transposed=True)
        return [*blocks, *transposed]
    if op == "product":
        return fma.grouped_gemm_fp8(fma.Fp8Blocks(*s["x"]), fma.Fp8Blocks(*s["w"]), s["M_array"], output_dtype=s["dtype"])
    if op == "linear":
        x, w = _leaf(s["x"]), _leaf(s["w"])
        y = fma.grouped_linear_fp8(x, w, s["M_array"])
        y.backward(s["dy"])
        return dict(y=y.detach(), x_grad=x.grad, w_grad=w.grad)
    if op == "swiglu":
        x = _leaf(s["x"])
        y = fma.swiglu_packed_fp8(x)
        y.backward(s["dy"])
        return dict(y=y.detach(), x_grad=x.grad)
    if op == "infer":
        with torch.no_grad():
            return fma.swiglu_experts_fp8(s["x"], s["gates"], s["selected"], fma.Fp8Blocks(*s["w1"]), fma.Fp8Blocks(*s["w2"]))
    x, gates, w1, w2 = (_leaf(s[n]) for n in ("x", "gates", "w1", "w2"))
    y = fma.swiglu_experts_fp8(x, gates, s["selected"], w1, w2)
    y.backward(s["dy"])
    return dict(y=y.detach(), x_grad=x.grad, gates_grad=gates.grad, w1_grad=w1.grad, w2_grad=w2.grad)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """bytes and operations of one pass: inputs read once, outputs written once; of the weights those of the experts that some row is
    for (their expected number at equal odds). A training step also writes every weight's gradient."""
    op, s = case["op"], BYTES[case["dtype"]]
    if op == "quantize":
        n = case["E"] * case["N"] * case["K"]
        return dict(bytes=n * (s + (1 if case["block_rows"] == 1 else 2)), flops=0)
    if op == "swiglu":
        return dict(bytes=case["R"] * case["I"] * s * 6, flops=0)  # x and dy in, y and dx out
    if op in ("product", "linear"):
        R, E, N, K = (case[n] for n in ("R", "E", "N", "K"))
        flops = 2 * R * N * K
        if op == "linear":
            return dict(bytes=s * (2 * R * (N + K) + 2 * E * N * K), flops=3 * flops)
        return dict(bytes=R * K + E * (1.0 - (1.0 - 1.0 / E) ** R) * N * K + R * N * s, flops=flops)
    T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
    flops = 2 * T * k * 3 * H * I
    if op == "train":
        return dict(bytes=s * (4 * T * H + 2 * E * 3 * H * I), flops=3 * flops)
    return dict(bytes=s * 2 * T * H + E * (1.0 - (1.0 - k / E) ** T) * 3 * H * I, flops=flops)


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------


def _exact_blocks(x, rows):
    """(values, scales) in 64 bits from x [N, K]; scales [n, k]"""
    N, K = x.shape
    n, k = -(-N // rows), -(-K // 128)
    full = torch.zeros(n * rows, k * 128, dtype=torch.float64, device=x.device)
    full[:N, :K] = x
    cells = full.view(n, rows, k, 128)
    fraction, exponent = torch.frexp(cells.abs().amax(dim=(1, 3)))  # 448 = 0.875 * 2^9
    scales = torch.exp2((exponent - 9 + (fraction > 0.875)).double().clamp(min=-126.0))
    scales[(fraction == 0)] = 2.0**-126
    v = cells / scales[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3.0)
    return (torch.round(v / step) * step).reshape(n * rows, k * 128)[:N, :K], scales


def _exact_seen(x, rows=1):
    values, scales = _exact_blocks(x, rows)
    return values * scales.repeat_interleave(rows, 0)[: x.shape[0]].repeat_interleave(128, 1)[:, : x.shape[1]]


def _exact_halves(h):
    return torch.cat([_exact_seen(half) for half in h.split(h.shape[1] // 2, 1)], 1)


def _exact_stored(blocks, rows):
    """the numbers that stored blocks [.., N, K] stand for, as a list of matrices"""
    values, scales = blocks
    matrices = []
    for v, s in zip(values.reshape(-1, *values.shape[-2:]), scales.reshape(-1, *scales.shape[-2:])):
        s = torch.exp2(s.view(torch.uint8).double() - 127.0)
        matrices.append(v.double() * s.repeat_interleave(rows, 0)[: v.shape[0]].repeat_interleave(128, 1)[:, : v.shape[1]])
    return matrices


def _exact_swiglu(h):
    up, gate = h.split(h.shape[1] // 2, 1)
    return up * gate / (1.0 + torch.exp(-gate))


def _exact_swiglu_grad(h, dy):
    up, gate = h.split(h.shape[1] // 2, 1)
    s = 1.0 / (1.0 + torch.exp(-gate))
    return torch.cat([dy * gate * s, dy * up * (s + gate * s * (1.0 - s))], 1)


def _exact_quantize(s):
    outputs = [[], [], [], []]
    for x in s["x"].double():
        values, scales = _exact_blocks(x, s["block_rows"])
        for out, v in zip(outputs, (values, scales, values.t(), scales.t())):
            out.append(v)
    outputs = [torch.stack(o) for o in outputs]
    for i in (1, 3):
        outputs[i] = torch.nn.functional.pad(outputs[i], (0, -outputs[i].shape[-1] % 4), value=1.0)
    return outputs[:2] if s["block_rows"] == 1 else outputs


def _exact_linear(s):
    w, dy, x = s["w"], s["dy"].double(), _exact_seen(s["x"].double())
    seen = _exact_seen(dy)
    y, x_grad, w_grad = [], [], []
    first = 0
    for e, n in enumerate(s["M_array"].view(torch.int32).tolist()):
        we, rows = _exact_seen(w[e].double(), 128), slice(first, first + n)
        y.append(x[rows] @ we.t())
        x_grad.append(seen[rows] @ we)
        w_grad.append(dy[rows].t() @ x[rows])
        first += n
    return dict(y=torch.cat(y), x_grad=torch.cat(x_grad), w_grad=torch.stack(w_grad))


def _exact_experts(s):
    training, gates, chosen = s["op"] == "train", s["gates"].double(), s["selected"].long()
    x = _exact_seen(s["x"].double())
    y, x_grad, gates_grad = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(gates)
    w1_grad, w2_grad = [], []
    stored = None if training else (_exact_stored(s["w1"], 128), _exact_stored(s["w2"], 128))
    for e in range(s["E"]):
        if training:
            half = s["w1"].shape[1] // 2
            w1 = torch.cat([_exact_seen(s["w1"][e, i * half : (i + 1) * half].double(), 128) for i in (0, 1)])
            w2 = _exact_seen(s["w2"][e].double(), 128)
        else:
            w1, w2 = torch.cat(stored[0][2 * e : 2 * e + 2]), stored[1][e]
        t, j = (chosen == e).nonzero(as_tuple=True)
        xe, ge = x[t], gates[t, j][:, None]
        h = xe @ w1.t()
        act = _exact_seen(_exact_swiglu(h))
        o = act @ w2.t()
        y.index_add_(0, t, o * ge)
        if not training:
            continue
        dy = s["dy"].double()[t]
        gates_grad[t, j] = (dy * o).sum(1)
        h_grad = _exact_swiglu_grad(_exact_halves(h), _exact_seen(dy * ge) @ w2)
        x_grad.index_add_(0, t, _exact_halves(h_grad) @ w1)
        w1_grad.append(h_grad.t() @ xe)
        w2_grad.append((dy * ge).t() @ act)
    if not training:
        return y
    return dict(y=y, x_grad=x_grad, gates_grad=gates_grad, w1_grad=torch.stack(w1_grad), w2_grad=torch.stack(w2_grad))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(s)
    if op == "product":
        x, y, first = _exact_stored(s["x"], 1)[0], [], 0
        for w, n in zip(_exact_stored(s["w"], 128), s["M_array"].view(torch.int32).tolist()):
            y.append(x[first : first + n] @ w.t())
            first += n
        return torch.cat(y)
    if op == "linear":
        return _exact_linear(s)
    if op == "swiglu":
        x = s["x"].double()
        return dict(y=_exact_swiglu(x), x_grad=_exact_swiglu_grad(_exact_halves(x), s["dy"].double()))
    return _exact_experts(s)
