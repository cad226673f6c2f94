"""The microscaled four-bit format (MXFP4): values in groups of 32 along the last axis, a group one power-of-two scale (E8M0) and
32 E2M1 codes. Unlike the framework's other formats it is one for activations too: a product of two matrices held in it runs on the
device's block-scaled matrix instructions (`ops.mxfp4_linear`, `mxfp4_moe.mxfp4_moe`), with no expansion of the weights.

The rounding of a group: scale 2^e with e = floor(log2 of the largest magnitude) - 2, not below -127; a value becomes the nearest of
0, 1/2, 1, 3/2, 2, 3, 4 and 6 times the scale, ties to the even code, beyond 6 to 6. A group that holds an infinity or a NaN
stands for NaN as a whole (scale byte 255, codes 0): the format has no other way to say so. No counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from hibana_amd import _lib

GROUP = 32
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # HB_BF16, HB_F16, HB_F32
CODES = 3  # HB_MXFP4


class Mxfp4(NamedTuple):
    """Values [..., K] held in the format."""
    codes: torch.Tensor   # uint8 [..., K / 2], element 2 i in the low nibble of byte i
    scales: torch.Tensor  # uint8 [..., K / 32], byte b for 2^(b - 127), 255 for NaN

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], self.codes.shape[-1] * 2)

    @property
    def device(self) -> torch.device:
        return self.codes.device


def check(q: Mxfp4, what: str) -> None:
    if q.codes.dtype != torch.uint8 or q.scales.dtype not in (torch.uint8, torch.float8_e8m0fnu) or q.codes.ndim == 0 or q.codes.shape[-1] % 16 or \
            q.scales.shape != (*q.codes.shape[:-1], q.codes.shape[-1] // 16):
        raise ValueError(f"{what}: codes uint8 [..., K / 2] and scales uint8 [..., K / 32], K a multiple of {GROUP}")


def flat(q: Mxfp4, what: str) -> Mxfp4:
    """The same values as whole rows, contiguous and on the boundaries the kernels read at (a copy only where they are not)."""
    check(q, what)
    k = q.codes.shape[-1]
    codes, scales = q.codes.reshape(-1, k).contiguous(), q.scales.view(torch.uint8).reshape(-1, k // 16).contiguous()
    return Mxfp4(codes if codes.data_ptr() % 16 == 0 else codes.clone(), scales)


def rows16(x: torch.Tensor) -> torch.Tensor:
    """x as contiguous rows that start on a 16-byte boundary."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def quantize(x: torch.Tensor) -> Mxfp4:
    """x [..., K] (BF16, FP16 or FP32; K a multiple of 32) rounded to the format."""
    kind = TYPES.get(x.dtype)
    if kind is None or x.ndim == 0 or x.shape[-1] % GROUP:
        raise ValueError(f"mxfp4.quantize: BF16, FP16 or FP32 [..., K], K a multiple of {GROUP}")
    _lib.need_one_gpu(x)
    shape, k = x.shape, x.shape[-1]
    codes = torch.empty((*shape[:-1], k // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*shape[:-1], k // GROUP), dtype=torch.uint8, device=x.device)
    if x.numel():
        xc = rows16(x)  # held until the launch is enqueued
        code = _lib.lib().hb_mxfp4_quantize(xc.data_ptr(), kind, x.numel() // k, k, codes.data_ptr(), scales.data_ptr(), _lib.stream())
        if code:
            _lib.check(code, "mxfp4.quantize")
    return Mxfp4(codes, scales)


def dequantize(q: Mxfp4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `q` stands for, [..., K]: exact in FP32 and in BF16; FP16 rounds what it does not hold."""
    kind = TYPES.get(dtype)
    if kind is None:
        raise ValueError("mxfp4.dequantize: to BF16, FP16 or FP32")
    check(q, "mxfp4.dequantize")
    _lib.need_one_gpu(q.codes, q.scales)
    out = torch.empty(q.shape, dtype=dtype, device=q.codes.device)
    if out.numel():
        f = flat(q, "mxfp4.dequantize")
        code = _lib.lib().hb_mxfp4_dequantize(f.codes.data_ptr(), f.scales.data_ptr(), f.codes.shape[0], q.shape[-1], kind, out.data_ptr(), _lib.stream())
        if code:
            _lib.check(code, "mxfp4.dequantize")
    return out


def tile(q: Mxfp4, gated: bool = False) -> torch.Tensor:
    """Weights [N, K] or stacked ones [E, N, K] in the layout the products read (csrc/mxfp4.hpp): uint8 [bytes] or [E, bytes].
    `gated`: fc1 of gated experts, rows [up; gate]."""
    check(q, "mxfp4.tile")
    if q.codes.ndim not in (2, 3) or not q.codes.numel():
        raise ValueError("mxfp4.tile: a matrix [N, K] or stacked matrices [E, N, K]")
    _lib.need_one_gpu(q.codes, q.scales)
    n, k = q.shape[-2:]
    size = _lib.lib().hb_mxfp4_tiled_bytes(n, k)
    if size == 0:
        raise ValueError(f"mxfp4.tile: a matrix [{n}, {k}] is past what the kernels index")
    tiled = torch.empty((*q.codes.shape[:-2], size), dtype=torch.uint8, device=q.codes.device)
    f = flat(q, "mxfp4.tile")
    lo = 0
    stacked = tiled.view(-1, size)
    while lo < stacked.shape[0]:  # a launch's grid holds 65535 matrices
        count = min(65535, stacked.shape[0] - lo)
        _lib.check(_lib.lib().hb_mxfp4_repack(f.codes[lo * n:].data_ptr(), f.scales[lo * n:].data_ptr(), count, n, k, int(gated), stacked[lo:].data_ptr(),
                                              _lib.stream()), "mxfp4.tile")
        lo += count
    return tiled


def untile(tiled: torch.Tensor, n: int, k: int, gated: bool = False) -> Mxfp4:
    """The inverse of `tile`."""
    size = _lib.lib().hb_mxfp4_tiled_bytes(n, k)
    if size == 0 or tiled.dtype != torch.uint8 or tiled.shape[-1] != size or not tiled.is_contiguous():
        raise ValueError(f"mxfp4.untile: not the layout of [{n}, {k}] matrices")
    _lib.need_one_gpu(tiled)
    lead, count = tiled.shape[:-1], tiled.numel() // size
    codes = torch.empty((*lead, n, k // 2), dtype=torch.uint8, device=tiled.device)
    scales = torch.empty((*lead, n, k // GROUP), dtype=torch.uint8, device=tiled.device)
    for lo in range(0, count, 65535):
        _lib.check(_lib.lib().hb_mxfp4_unpack(tiled.view(count, size)[lo:].data_ptr(), min(65535, count - lo), n, k, int(gated), codes.view(count, n, -1)[lo:].data_ptr(),
                                              scales.view(count, n, -1)[lo:].data_ptr(), _lib.stream()), "mxfp4.untile")
    return Mxfp4(codes, scales)
