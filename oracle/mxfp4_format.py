"""The microscaled four-bit format in FP64 (CPU, torch): the rounding by the borders between neighbouring values, the values back,
the products and the routed experts on them, straight from their definitions. What the tests compare the kernels with, never the product."""
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


def between(lo: torch.Tensor, hi: torch.Tensor):
    """The smallest and the largest magnitude that the rounding of values with magnitudes lo .. hi [..., K] can give (a group's scale is
    that of its largest: of lo's or of hi's, or equal for both)."""
    def under(v, scale_of):
        _, e = torch.frexp(scale_of.reshape(*v.shape[:-1], -1, GROUP).amax(-1))
        unit = torch.ldexp(torch.ones(e.shape, dtype=torch.float64), (e - 3).clamp(min=-127)).repeat_interleave(GROUP, -1)
        a = v / unit
        code = (a > 0.25).long() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
        return LEVELS[code] * unit
    every = torch.stack([under(v, s) for v in (lo, hi) for s in (lo, hi)])
    return every.amin(0), every.amax(0)


def moe_pairs(x, ids, fc1, fc2, base: int = 0):
    """FP64 [M, k, H_out] twice: each pair's expert output (zero where the id is not one of base .. base + E - 1), and how far one
    computed with FP32 sums may be from it. fc1 / fc2: (codes, scales) stacked; gated (fc1 of 2 I rows, [up; gate]) or ReLU^2.

    An FP32 sum of K products is off by at most K 2^-24 sum |x w|; silu moves by at most 1.1 times its argument's change, and is
    off by 2^-20 of its value at most where it is computed. That moves h, and where it moves a value of h over a border between two codes, the
    product's operand."""
    m, k = ids.shape
    experts, inter = fc2[0].shape[0], 2 * fc2[0].shape[2]
    xq = through(x)
    out, off = (torch.zeros(m, k, fc2[0].shape[1], dtype=torch.float64) for _ in range(2))
    for e in sorted(set(ids.flatten().tolist())):
        if not base <= e < base + experts:
            continue
        row, slot = torch.nonzero(ids == e, as_tuple=True)
        w1, w2 = dequantize(fc1[0][e - base], fc1[1][e - base]), dequantize(fc2[0][e - base], fc2[1][e - base])
        y = xq[row] @ w1.T
        dy = w1.shape[1] * 2.0 ** -24 * (xq[row].abs() @ w1.abs().T)
        if w1.shape[0] == 2 * inter:
            up, gate, dup, dgate = y[:, :inter], y[:, inter:], dy[:, :inter], dy[:, inter:]
            silu = gate / (1.0 + torch.exp(-gate))
            h = silu * up
            dh = 1.1 * dgate * (up.abs() + dup) + silu.abs() * dup + 2.0 ** -20 * h.abs()
        else:
            h = y.clamp(min=0) ** 2
            dh = 2 * y.clamp(min=0) * dy + dy ** 2 + 2.0 ** -24 * h
        hq = through(h)
        least, most = between((h.abs() - dh).clamp(min=0), h.abs() + dh)
        spread = torch.maximum(hq.abs() - least, most - hq.abs())
        spread = spread + torch.where(dh >= h.abs(), most, torch.zeros_like(most))  # (a value that may be of the other sign)
        out[row, slot] = hq @ w2.T
        off[row, slot] = spread @ w2.abs().T + inter * 2.0 ** -24 * ((hq.abs() + spread) @ w2.abs().T)
    return out, off


def moe(x, ids, weights, fc1, fc2, base: int = 0):
    """FP64 [M, H_out] twice: the weighted sum of a row's pairs, and how far an FP32 one may be from it ahead of its last rounding."""
    y, off = moe_pairs(x, ids, fc1, fc2, base)
    w = torch.where((ids >= base) & (ids < base + fc2[0].shape[0]), weights.double(), torch.zeros(ids.shape, dtype=torch.float64))[..., None]
    return (y * w).sum(1), (off * w.abs()).sum(1) + (ids.shape[1] + 1) * 2.0 ** -24 * (y * w).abs().sum(1)
