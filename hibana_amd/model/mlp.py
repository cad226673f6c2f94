"""The dense SwiGLU MLP behind the reference's `Mlp.__call__` (hibana/model/mlp.py:26-48): gate|up and down as NVFP4
linears, each with an optional 3-bit decode copy.

    gate_up = nvfp4_linear(x, gate_up)                         (its 3-bit copy at decode sizes, weight-only)
    3-bit decode of both:    the two lines around this one in one call, `w3.w3_mlp`
    3-bit decode of `down`:  x_q, s = silu_mul_quant_groups(gate_up, pairs, torch_chain=True);  w3_linear(x_q, down.w3, s)
    otherwise:               nvfp4_linear(silu_and_mul(gate_up, pairs), down)

With both linears in the microscaled four-bit format (`Mxfp4Linear`) the activations are four bits wide too, rounded on the way into each
product: mxfp4_linear(silu_mul_quant_mxfp4(mxfp4_linear(x, gate_up), pairs), down).

With `adapters`, a pool beside each linear (or None), and a call's `index`, each row's own adapter is added to both products
(`adapters.add`), which are then calls of their own; rows without an adapter have the bits that they have without an `index`. A pool of the down
projection reads the SiLU product in BF16 where its linear reads that or (3-bit decode) the groups rounded from it, and the microscaled
format's own rows, rounded to four bits, where its linear reads those. A serving
form: no gradient is recorded, of the rows or of pools that take one.

Assembled from linears already loaded. The reference's NVFP4 activation paths (`prequantized`, the fused prefill
gate/up GEMM that rounds SiLU(gate) * up to NVFP4 in its epilogue) have no counterpart: the NVFP4 kernels here are
weight-only.
"""
from __future__ import annotations

import torch

from hibana_amd.kernels import adapters as low_rank, mxfp4, ops, w3
from hibana_amd.weights.mxfp4 import Mxfp4Linear


class Mlp:
    def __init__(self, gate_up, down, adapters=None):
        """gate_up: `Nvfp4Linear` (or `Mxfp4Linear`, `down` then too) [2 I, H], rows [gate; up] or interleaved in blocks of `gate_up.pairs`; down [H, I].
        adapters: (of gate_up, of down), each an `Adapters` of that projection (its b's columns in gate_up's order of rows) or None."""
        if gate_up.out_features != 2 * down.in_features or down.out_features != gate_up.in_features:
            raise ValueError("gate_up [2 I, H] and down [H, I] do not describe one MLP")
        if isinstance(gate_up, Mxfp4Linear) != isinstance(down, Mxfp4Linear):
            raise ValueError("Mlp: one linear in the microscaled four-bit format, the other not")
        self.gate_up, self.down = gate_up, down
        self.adapters = (None, None) if adapters is None else tuple(adapters)
        if len(self.adapters) != 2 or any(pool is not None and (pool.in_features, pool.out_features) != (lin.in_features, lin.out_features)
                                          for pool, lin in zip(self.adapters, (gate_up, down))):
            raise ValueError("Mlp: adapters of the two projections, or None for one without")

    def __call__(self, x: torch.Tensor, prequantized=None, index: torch.Tensor | None = None) -> torch.Tensor:
        """x [rows, H] BF16 -> BF16 [rows, H]; on `Mxfp4Linear`s also FP16 or FP32, the result of that type, or rows already rounded
        (`mxfp4.Mxfp4`), the result BF16. `index` int32 or int64 [rows]: each row's adapter (-1: none); without it no adapter is added."""
        if prequantized is not None:
            raise ValueError("Mlp: NVFP4 activations are not taken by the weight-only kernels")
        if index is not None and any(pool is not None for pool in self.adapters):
            return self._adapted(x, index)
        pairs = self.gate_up.pairs
        if isinstance(self.gate_up, Mxfp4Linear):
            gate_up = ops.mxfp4_linear(x, self.gate_up)
            return ops.mxfp4_linear(ops.silu_mul_quant_mxfp4(gate_up, pairs), self.down, gate_up.dtype)
        if x.ndim == 2 and ops.w3_decode(self.gate_up, x.shape[0]) and ops.w3_decode(self.down, x.shape[0]) and \
                w3.w3_mlp_takes(x, self.gate_up.w3, self.down.w3):
            return w3.w3_mlp(x, self.gate_up.w3, self.down.w3, pairs)
        gate_up = ops.nvfp4_linear(x, self.gate_up)
        if ops.w3_decode(self.down, gate_up.shape[0]):
            return self._down_in_three_bits(gate_up)
        return ops.nvfp4_linear(ops.silu_and_mul(gate_up, pairs), self.down)

    def _down_in_three_bits(self, gate_up: torch.Tensor) -> torch.Tensor:
        """3-bit decode: the SiLU product in BF16 rounded per 32-group for the 3-bit GEMM, in one launch."""
        x_q, x_scale = ops.silu_mul_quant_groups(gate_up, self.gate_up.pairs, torch_chain=True)
        return w3.w3_linear(x_q, self.down.w3, x_scale)

    def _adapted(self, x: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
        if not isinstance(x, torch.Tensor):
            raise ValueError("Mlp: adapters read rows as they are, not rounded ones")

        def add(y, rows, pool):
            with torch.no_grad():
                return y if pool is None else low_rank.add(y, rows, pool, index, out=y)
        pairs = self.gate_up.pairs
        if isinstance(self.gate_up, Mxfp4Linear):
            gate_up = add(ops.mxfp4_linear(x, self.gate_up), x, self.adapters[0])
            rounded = ops.silu_mul_quant_mxfp4(gate_up, pairs)
            y = ops.mxfp4_linear(rounded, self.down, gate_up.dtype)
            return y if self.adapters[1] is None else add(y, mxfp4.dequantize(rounded, gate_up.dtype), self.adapters[1])
        gate_up = add(ops.nvfp4_linear(x, self.gate_up), x, self.adapters[0])
        if ops.w3_decode(self.down, gate_up.shape[0]):  # the groups that it reads without adapters too
            y = self._down_in_three_bits(gate_up)
            return y if self.adapters[1] is None else add(y, ops.silu_and_mul(gate_up, pairs), self.adapters[1])
        h = ops.silu_and_mul(gate_up, pairs)
        return add(ops.nvfp4_linear(h, self.down), h, self.adapters[1])
