"""The microscaled four-bit format in FP64 (CPU, torch): the rounding by the borders between neighbouring values, the values back,
the products and the routed experts on them, straight from their definitions. The checker of the MXFP4 kernels, never the product."""
from __future__ import annotations

import torch

GROUP = 32
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x: torch.Tensor):
    """[..., K] -> (codes uint8 [..., K / 2], scale bytes uint8 [..., K / 32])."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    top = g.abs().amax(-1)
    finite = torch.isfinite(g).all(-1) & (top < 2.0 ** 128)
    top = torch.where(finite, top, torch.zeros_like(top))
    _, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1
    byte = torch.where(top == 0, torch.zeros_like(e), (e - 1 - 2 + 127).clamp(min=0))
    v = torch.where(finite[..., None], g, torch.zeros_like(g)) / torch.ldexp(torch.ones_like(top), byte - 127)[..., None]
    a = v.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code + 8 * torch.signbit(v)).reshape(x.shape)
    code = torch.where(finite[..., None].expand_as(g).reshape(x.shape), code, torch.zeros_like(code)).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(finite, byte, torch.full_like(byte, 255)).to(torch.uint8)


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """FP64 [..., K]."""
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    value = torch.cat((LEVELS, -LEVELS))[nibbles]
    unit = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales.int() - 127)
    unit = torch.where(scales == 255, torch.full_like(unit, float("nan")), unit)
    return value * unit.repeat_interleave(GROUP, dim=-1)


def through(x: torch.Tensor) -> torch.Tensor:
    return dequantize(*quantize(x))


def silu_mul(gate_up: torch.Tensor, pairs: int = 0) -> torch.Tensor:
    """FP64 silu(gate) * up of [..., 2 I]."""
    x = gate_up.double()
    half = x.shape[-1] // 2
    both = x.reshape(*x.shape[:-1], -1, 2, pairs or half)
    gate, up = both[..., 0, :].reshape(*x.shape[:-1], half), both[..., 1, :].reshape(*x.shape[:-1], half)
    return gate / (1.0 + torch.exp(-gate)) * up


def moe_pairs(x, ids, fc1, fc2, base: int = 0):
    """FP64 [M, k, H_out]: each pair's expert output, zero where the id is not one of base .. base + E - 1. fc1 / fc2: (codes, scales)
    stacked; gated (fc1 of 2 I rows, [up; gate]) or ReLU^2."""
    m, k = ids.shape
    experts, inter = fc2[0].shape[0], 2 * fc2[0].shape[2]
    xq = through(x)
    out = torch.zeros(m, k, fc2[0].shape[1], dtype=torch.float64)
    for e in sorted(set(ids.flatten().tolist())):
        if not base <= e < base + experts:
            continue
        row, slot = torch.nonzero(ids == e, as_tuple=True)
        y = xq[row] @ dequantize(fc1[0][e - base], fc1[1][e - base]).T
        h = y[:, inter:] / (1.0 + torch.exp(-y[:, inter:])) * y[:, :inter] if fc1[0].shape[1] == 2 * inter else y.clamp(min=0) ** 2
        out[row, slot] = through(h) @ dequantize(fc2[0][e - base], fc2[1][e - base]).T
    return out


def moe(x, ids, weights, fc1, fc2, base: int = 0) -> torch.Tensor:
    """FP64 [M, H_out]: the weighted sum of a row's pairs."""
    pairs = moe_pairs(x, ids, fc1, fc2, base)
    named = (ids >= base) & (ids < base + fc2[0].shape[0])
    return torch.where(named[..., None], pairs * weights.double()[..., None], torch.zeros_like(pairs)).sum(1)
