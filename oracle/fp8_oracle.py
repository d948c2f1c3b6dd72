"""64-bit oracle of the 8-bit block format and of the operators on it: the definition, element by element, on the CPU."""

import torch

BLOCK = 128
E4M3_MAX = 448.0


def scale_columns(K: int) -> int:
    return (K + 511) // 512 * 4


def quantize(x: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """x [N, K] -> (values float64 [N, K], scale bytes uint8 [ceil(N / block_rows), scale_columns(K)])"""
    x = x.double()
    N, K = x.shape
    n, k = -(-N // block_rows), -(-K // BLOCK)
    values = torch.zeros(N, K, dtype=torch.float64)
    scales = torch.full((n, scale_columns(K)), 127, dtype=torch.uint8)
    for i in range(n):
        rows = slice(i * block_rows, min(N, (i + 1) * block_rows))
        for j in range(k):
            columns = slice(j * BLOCK, min(K, (j + 1) * BLOCK))
            block = x[rows, columns]
            if not bool(torch.isfinite(block).all()):
                values[rows, columns] = float("nan")
                scales[i, j] = 255
                continue
            amax = float(block.abs().max()) if block.numel() else 0.0
            exponent = -126
            while amax > E4M3_MAX * 2.0**exponent:
                exponent += 1
            values[rows, columns] = round_e4m3(block * 2.0**-exponent)
            scales[i, j] = exponent + 127
    return values, scales


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """to the nearest multiple of the step at v's magnitude (2^-9 below 2^-6), ties to even; |v| <= 448"""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3.0)
    return torch.round(v / step) * step


def dequantize(values: torch.Tensor, scales: torch.Tensor, block_rows: int = 1) -> torch.Tensor:
    N, K = values.shape
    s = torch.exp2(scales.view(torch.uint8).double() - 127.0)
    s = torch.where(scales.view(torch.uint8) == 255, torch.nan, s)
    return values.double() * s.repeat_interleave(block_rows, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]


def seen(x: torch.Tensor, block_rows: int = 1) -> torch.Tensor:
    return dequantize(*quantize(x, block_rows), block_rows)


def halves(h: torch.Tensor) -> torch.Tensor:
    I = h.size(1) // 2
    return torch.cat([seen(h[:, :I]), seen(h[:, I:])], 1)


def swiglu(h: torch.Tensor) -> torch.Tensor:
    up, gate = h.double().chunk(2, 1)
    return up * gate * torch.sigmoid(gate)


def swiglu_grad(h: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    up, gate = h.double().chunk(2, 1)
    s = torch.sigmoid(gate)
    return torch.cat([dy * gate * s, dy * up * (s + gate * s * (1 - s))], 1)
