"""The microscaled four-bit format (MXFP4): values in groups of 32 along the last axis, a group one power-of-two scale (E8M0) and
32 E2M1 codes. Unlike the framework's other formats it is one for activations too: a product of two matrices held in it runs on the
device's block-scaled matrix instructions (`ops.mxfp4_linear`, `mxfp4_moe.mxfp4_moe`), with no expansion of the weights.

The rounding of a group: scale 2^e with e = floor(log2 of the largest magnitude) - 2, not below -127; a value becomes the nearest of
0, 1/2, 1, 3/2, 2, 3, 4 and 6 times the scale, ties to the even code, beyond 6 to 6. A group that holds an infinity or a NaN
stands for NaN as a whole (scale byte 255, codes 0): the format has no other way to say so. No counterpart in the reference.
"""
from __future__ import annotations

import torch

from hibana_amd import _lib

GROUP = 32
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # HB_BF16, HB_F16, HB_F32
CODES = 3  # HB_MXFP4


class Mxfp4:
    """Values [..., K] held in the format: `codes` uint8 [..., K / 2], element 2 i in the low nibble of byte i, and `scales` uint8
    [..., K / 32], byte b for 2^(b - 127), 255 for NaN. Unpacks into the two. What a kernel here has rounded lies in one allocation, codes first,
    and becomes the two tensors when they are asked for: a small call pays for one."""
    __slots__ = ("_codes", "_scales", "_block", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        self._codes, self._scales, self._block = codes, scales, None
        self.shape = (*codes.shape[:-1], codes.shape[-1] * 2) if codes.ndim else ()

    @classmethod
    def of_block(cls, block: torch.Tensor, shape: tuple[int, ...]) -> "Mxfp4":
        """Codes and scales one behind the other in `block`."""
        self = cls.__new__(cls)
        self._codes = self._scales = None
        self._block, self.shape = block, shape
        return self

    def _split(self) -> None:
        *lead, k = self.shape
        size = self._block.numel() * 16 // 17  # 16 bytes of codes to one of scales
        self._codes = self._block[:size].view(*lead, k // 2)
        self._scales = self._block[size:].view(*lead, k // GROUP)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._split()
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._split()
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._codes if self._block is None else self._block).device

    def __iter__(self):
        return iter((self.codes, self.scales))

    def __reduce__(self):
        return Mxfp4, (self.codes, self.scales)


def check(q: Mxfp4, what: str) -> None:
    codes, scales = q
    if codes.dtype != torch.uint8 or scales.dtype not in (torch.uint8, torch.float8_e8m0fnu) or codes.ndim == 0 or codes.shape[-1] % 16 or \
            scales.shape != (*codes.shape[:-1], codes.shape[-1] // 16):
        raise ValueError(f"{what}: codes uint8 [..., K / 2] and scales uint8 [..., K / 32], K a multiple of {GROUP}")


def flat(q: Mxfp4, what: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales as whole rows, contiguous and on the boundaries the kernels read at (a copy only where they are not)."""
    check(q, what)
    k = q.codes.shape[-1]
    codes, scales = q.codes.reshape(-1, k).contiguous(), q.scales.view(torch.uint8).reshape(-1, k // 16).contiguous()
    return codes if codes.data_ptr() % 16 == 0 else codes.clone(), scales


def places(q: Mxfp4, what: str):
    """(address of the codes, address of the scales, what to hold until the launch that reads them is enqueued, the current stream), on the
    current device."""
    block = q._block
    if block is not None:
        stream = _lib.stream_of(block)
        at = block.data_ptr()
        return at, at + block.numel() * 16 // 17, block, stream
    check(q, what)
    stream = _lib.stream_of(q.codes, q.scales)
    held = flat(q, what)
    return held[0].data_ptr(), held[1].data_ptr(), held, stream


def rows16(x: torch.Tensor) -> torch.Tensor:
    """x as contiguous rows that start on a 16-byte boundary."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def quantize(x: torch.Tensor) -> Mxfp4:
    """x [..., K] (BF16, FP16 or FP32; K a multiple of 32) rounded to the format."""
    kind = TYPES.get(x.dtype)
    shape = tuple(x.shape)
    if kind is None or not shape or shape[-1] % GROUP:
        raise ValueError(f"mxfp4.quantize: BF16, FP16 or FP32 [..., K], K a multiple of {GROUP}")
    stream = _lib.stream_of(x)
    n = x.numel()
    block = x.new_empty(n // GROUP * 17, dtype=torch.uint8)
    if n:
        xc = rows16(x)  # held until the launch is enqueued
        at = block.data_ptr()
        code = _lib.lib().hb_mxfp4_quantize(xc.data_ptr(), kind, n // shape[-1], shape[-1], at, at + n // 2, stream)
        if code:
            _lib.check(code, "mxfp4.quantize")
    return Mxfp4.of_block(block, shape)


def dequantize(q: Mxfp4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `q` stands for, [..., K]: exact in FP32 and in BF16; FP16 rounds what it does not hold."""
    kind = TYPES.get(dtype)
    if kind is None:
        raise ValueError("mxfp4.dequantize: to BF16, FP16 or FP32")
    codes, scales, held, stream = places(q, "mxfp4.dequantize")
    out = (q._codes if q._block is None else q._block).new_empty(q.shape, dtype=dtype)
    n = out.numel()
    if n:
        k = q.shape[-1]
        code = _lib.lib().hb_mxfp4_dequantize(codes, scales, n // k, k, kind, out.data_ptr(), stream)
        if code:
            _lib.check(code, "mxfp4.dequantize")
    return out


def tile(q: Mxfp4, gated: bool = False) -> torch.Tensor:
    """Weights [N, K] or stacked ones [E, N, K] in the layout the products read (csrc/mxfp4.hpp): uint8 [bytes] or [E, bytes].
    `gated`: fc1 of gated experts, rows [up; gate]. It is there when this returns: a call that finds the weights not laid out does it on its own stream
    without its caller knowing, and the next call may be another stream's; nor does anything read the codes then, which may be released."""
    check(q, "mxfp4.tile")
    if q.codes.ndim not in (2, 3) or not q.codes.numel():
        raise ValueError("mxfp4.tile: a matrix [N, K] or stacked matrices [E, N, K]")
    _lib.need_one_gpu(q.codes, q.scales)
    if torch.cuda.is_current_stream_capturing():  # it would lie in the graph's memory, and hold nothing before a replay
        raise RuntimeError("mxfp4.tile: weights are laid out ahead of a capture")
    n, k = q.shape[-2:]
    size = _lib.lib().hb_mxfp4_tiled_bytes(n, k)
    if size == 0:
        raise ValueError(f"mxfp4.tile: a matrix [{n}, {k}] is past what the kernels index")
    tiled = torch.empty((*q.codes.shape[:-2], size), dtype=torch.uint8, device=q.codes.device)
    codes, scales = flat(q, "mxfp4.tile")
    lo = 0
    stacked = tiled.view(-1, size)
    while lo < stacked.shape[0]:  # a launch's grid holds 65535 matrices
        count = min(65535, stacked.shape[0] - lo)
        _lib.check(_lib.lib().hb_mxfp4_repack(codes[lo * n:].data_ptr(), scales[lo * n:].data_ptr(), count, n, k, int(gated), stacked[lo:].data_ptr(),
                                              _lib.stream()), "mxfp4.tile")
        lo += count
    torch.cuda.current_stream().synchronize()  # once a matrix
    return tiled


def check_tiled(tiled: torch.Tensor | None, shape: tuple[int, ...], what: str) -> None:
    """That `tiled` has the layout's bytes for matrices of `shape` ([N, K] or [E, N, K])."""
    size = _lib.lib().hb_mxfp4_tiled_bytes(*shape[-2:])
    if tiled is None or size == 0 or tiled.dtype != torch.uint8 or tuple(tiled.shape) != (*shape[:-2], size) or not tiled.is_contiguous() or tiled.data_ptr() % 16:
        raise ValueError(f"{what}: not the layout of {list(shape)}")


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
