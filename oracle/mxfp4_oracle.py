"""MXFP4 in 64 bits, from its definition: blocks of 32 e2m1 codes with a shared power of two (test infrastructure, CPU)."""
import torch

BLOCK = 32
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantize(a: torch.Tensor):
    """Rows [.., K] -> packed codes [.., K / 2], scale bytes [.., K / 32]: the nearest value of each block's grid, ties to even codes."""
    blocks = a.double().unflatten(-1, (-1, BLOCK))
    largest = blocks.abs().amax(-1)
    special = ~torch.isfinite(blocks).all(-1)
    largest = torch.where(special, torch.ones_like(largest), largest)
    _, exponent = torch.frexp(largest)                       # largest = f 2^exponent, f in [0.5, 1)
    power = torch.where(largest == 0, torch.full_like(exponent, -127), (exponent - 1 - 2).clamp(min=-127))
    v = torch.where(special[..., None], torch.zeros_like(blocks), blocks) / torch.exp2(power.double())[..., None]
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64)
    code = torch.zeros(v.shape, dtype=torch.uint8)
    for c in range(1, 8):
        middle = (grid[c - 1] + grid[c]) / 2
        code[(v.abs() >= middle) if c % 2 == 0 else (v.abs() > middle)] = c
    code |= torch.signbit(v).to(torch.uint8) << 3
    code[special] = 0
    code = code.flatten(-2)
    scale = torch.where(special, torch.full_like(power, 255), power + 127).to(torch.uint8)
    return code[..., ::2] | (code[..., 1::2] << 4), scale


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What packed codes and scale bytes stand for, fp64."""
    codes, scales = codes.cpu().view(torch.uint8), scales.cpu().view(torch.uint8)
    grid = torch.tensor(MAGNITUDES + [-m for m in MAGNITUDES], dtype=torch.float64)
    v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2)
    power = torch.exp2(scales.double() - 127)
    power[scales == 255] = float("nan")
    return (v.unflatten(-1, (-1, BLOCK)) * power[..., None]).flatten(-2)


def product(xq, wq, xs, ws, bias=None):
    """X W^T + bias and, for error bounds, |X| |W|^T."""
    x, w = values(xq, xs), values(wq, ws)
    y = x.reshape(-1, x.shape[-1]) @ w.t()
    size = x.abs().reshape(-1, x.shape[-1]) @ w.abs().t()
    if bias is not None:
        y = y + bias.double().cpu()
        size = size + bias.double().cpu().abs()
    return y, size


def gated(xq, wq, xs, ws):
    """silu(X Wg^T) * (X Wu^T), with both factors and their |X| |W|^T."""
    y, size = product(xq, wq, xs, ws)
    n = wq.shape[0] // 2
    gate, up = y[:, :n], y[:, n:]
    return gate * torch.sigmoid(gate) * up, (gate, up, size[:, :n], size[:, n:])
