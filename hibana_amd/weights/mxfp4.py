"""A linear whose weights are held in the microscaled four-bit format (kernels/mxfp4.py): E2M1 codes two a byte and one E8M0 scale for
32 weights along K, as checkpoints of the format store them, or rounded here from a dense matrix. `tile()` lays them out once for the
kernels. Its product takes four-bit activations too: `ops.mxfp4_linear`. The `Linear` protocol's `w3` is never set: such a linear
has no three-bit copy.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from hibana_amd.kernels import mxfp4


@dataclass
class Mxfp4Linear:
    codes: torch.Tensor | None   # uint8 [N, K / 2]
    scales: torch.Tensor | None  # uint8 [N, K / 32] (or float8_e8m0fnu)
    pairs: int = 0               # an MLP's gate | up: rows alternate in blocks of this many (0: [gate; up])
    tiled: torch.Tensor | None = None  # the kernels' layout (built by tile())
    out_features: int = 0
    in_features: int = 0
    w3: object = None
    rooms: dict = field(default_factory=dict, init=False, repr=False, compare=False)  # the workspace a call of (rows, type) takes

    def __post_init__(self):
        if self.codes is not None:
            mxfp4.check(self.held, "Mxfp4Linear")
            if self.codes.ndim != 2 or not self.codes.numel():
                raise ValueError("Mxfp4Linear: codes uint8 [N, K / 2]")
            self.out_features, self.in_features = self.codes.shape[0], 2 * self.codes.shape[1]
        if self.tiled is not None or self.codes is None:
            mxfp4.check_tiled(self.tiled, (self.out_features, self.in_features), "Mxfp4Linear")

    @classmethod
    def from_dense(cls, weight: torch.Tensor, pairs: int = 0) -> "Mxfp4Linear":
        """weight [N, K] BF16, FP16 or FP32, rounded to the format."""
        return cls(*mxfp4.quantize(weight), pairs=pairs)

    @property
    def held(self) -> mxfp4.Mxfp4:
        """Codes and scales by rows; from the kernels' layout where only that is left."""
        if self.codes is None:
            return mxfp4.untile(self.tiled, self.out_features, self.in_features)
        return mxfp4.Mxfp4(self.codes, self.scales)

    @property
    def bytes(self) -> int:
        return self.out_features * self.in_features * 17 // 32

    def tile(self, release: bool = False) -> "Mxfp4Linear":
        """Build the kernels' layout (once); `release` drops the codes and scales by rows."""
        if self.tiled is None:
            self.tiled = mxfp4.tile(self.held)
        if release:
            self.codes = self.scales = None
        return self

    def dequantize(self) -> torch.Tensor:
        """FP32 [N, K]."""
        return mxfp4.dequantize(self.held)

    def __call__(self, x) -> torch.Tensor:
        from hibana_amd.kernels import ops
        return ops.mxfp4_linear(x, self)
