"""Low-rank adapters beside a shared projection and their gradients, in 64 bits, an adapter at a time, with the bounds on what a kernel
of FP32 sums may be off by."""
from __future__ import annotations

import torch

SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def _each(a, b, scale, ranks, index):
    """(rows, adapter, a, b, scale) of the adapters that rows have."""
    for i in range(a.shape[0]):
        rows = torch.nonzero(index == i).squeeze(1)
        r = a.shape[1] if ranks is None else int(ranks[i])
        if len(rows) and r:
            yield rows, i, a[i, :r].double(), b[i, :r].double(), 1.0 if scale is None else float(scale[i])


def add(y, x, a, b, scale, ranks, index):
    out = y.double().clone()
    for rows, _, ai, bi, s in _each(a, b, scale, ranks, index):
        out[rows] += s * (x[rows].double() @ ai.T) @ bi
    return out


def grads(dy, x, a, b, scale, ranks, index):
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    da, db = torch.zeros(a.shape, dtype=torch.float64, device=x.device), torch.zeros(b.shape, dtype=torch.float64, device=x.device)
    for rows, i, ai, bi, s in _each(a, b, scale, ranks, index):
        xr, dyr = x[rows].double(), dy[rows].double()
        g = s * dyr @ bi.T
        dx[rows] = g @ ai
        da[i, :len(ai)] = g.T @ xr
        db[i, :len(bi)] = s * (xr @ ai.T).T @ dyr
    return dx, da, db


def _two(length, terms, parts):
    """What a product of a product may be off by, relative to the same product of all the magnitudes: `length` FP32 additions of the inner sums, their
    cut into parts, `terms` additions of the outer ones. An addition is counted at 2^-23: the matrix instructions' own sums need not round to nearest."""
    return (length + 40) * 2.0 ** -23 + parts + (terms + 8) * 2.0 ** -23


# FP32 inner sums as operands, in three parts of the type: BF16 cut to 8 bits each, all of the 24; FP16 rounded to 11 bits each (2^-33), of values brought
# below 2^15, whose own smallest step is 2^-24: each of the three parts may be off by 2^-25 where it is brought down to a larger unit, the last one by its
# rounding too, 4 * 2^-25 / 2^14 of the largest
PARTS = {torch.bfloat16: 2.0 ** -24, torch.float16: 2.0 ** -33, torch.float32: 0.0}
LARGEST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -37, torch.float32: 0.0}


def add_bound(y, x, a, b, scale, ranks, index):
    """Element by element: one rounding of the result and the FP32 sums' errors."""
    dtype = y.dtype
    bound = torch.zeros(y.shape, dtype=torch.float64, device=x.device)
    for rows, _, ai, bi, s in _each(a, b, scale, ranks, index):
        inner = x[rows].double().abs() @ ai.abs().T
        rel = _two(x.shape[1], 3 * len(ai), PARTS[dtype])
        bound[rows] = abs(s) * (rel * (inner @ bi.abs()) + LARGEST[dtype] * inner.amax(1, keepdim=True) * bi.abs().sum(0))
    out = add(y, x, a, b, scale, ranks, index)
    return bound + (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * (out.abs() + bound) + SMALLEST[dtype]


def grads_bound(dy, x, a, b, scale, ranks, index):
    dtype = x.dtype
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    da, db = torch.zeros(a.shape, dtype=torch.float64, device=x.device), torch.zeros(b.shape, dtype=torch.float64, device=x.device)
    for rows, i, ai, bi, s in _each(a, b, scale, ranks, index):
        xr, dyr, m = x[rows].double().abs(), dy[rows].double().abs(), len(rows)
        g, h = abs(s) * dyr @ bi.abs().T, abs(s) * xr @ ai.abs().T
        dx[rows] = _two(dy.shape[1], 3 * len(ai), PARTS[dtype]) * (g @ ai.abs()) + LARGEST[dtype] * g.amax(1, keepdim=True) * ai.abs().sum(0)
        # (sums over rows: an adapter's largest value is the unit of all of its rows in FP16)
        da[i, :len(ai)] = _two(dy.shape[1], 3 * m, PARTS[dtype]) * (g.T @ xr) + LARGEST[dtype] * g.max() * xr.sum(0)
        db[i, :len(bi)] = _two(x.shape[1], 3 * m, PARTS[dtype]) * (h.T @ dyr) + LARGEST[dtype] * h.max() * dyr.sum(0)
    want = grads(dy, x, a, b, scale, ranks, index)
    return (dx + (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * (want[0].abs() + dx) + SMALLEST[dtype],
            da + 2.0 ** -22 * want[1].abs() + 2.0 ** -149, db + 2.0 ** -22 * want[2].abs() + 2.0 ** -149)
