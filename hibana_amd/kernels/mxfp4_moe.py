"""Routed experts whose weights and activations are both in the microscaled four-bit format (kernels/mxfp4.py), beside `w3_moe`:

    xq = x rounded to the format;  for each routed pair   h = silu(gate xq) * (up xq)  or  relu(up xq)^2   (FP32, then rounded to it)
    out = sum_k w_k down h_k                                                                              (FP32, rounded once)

fc1 [E, 2 I, H] with rows [up; gate] (gated) or [E, I, H] (ReLU^2), fc2 [E, H_out, I]; H and I multiples of 32. Deterministic,
graph-capturable, any number of rows (past 2^18 pairs in passes). No counterpart in the reference.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from hibana_amd import _lib
from hibana_amd.kernels import mxfp4

ID_TYPES = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)
MAX_EXPERTS = 960  # of one object: a plan's counts of them lie in LDS


@dataclass
class Mxfp4Experts:
    fc1_codes: torch.Tensor | None   # uint8 [E, 2 I or I, H / 2]
    fc1_scales: torch.Tensor | None  # uint8 [E, 2 I or I, H / 32]
    fc2_codes: torch.Tensor | None   # uint8 [E, H_out, I / 2]
    fc2_scales: torch.Tensor | None
    base: int = 0                    # the first expert's id
    tiled1: torch.Tensor | None = None  # the kernels' layout of the stacks (built by tile())
    tiled2: torch.Tensor | None = None
    shape1: tuple[int, int, int] | None = None  # (E, N1, H) and (E, H_out, I): kept when the tensors by rows are released
    shape2: tuple[int, int, int] | None = None

    def __post_init__(self):
        if self.shape1 is None:
            for codes, scales in ((self.fc1_codes, self.fc1_scales), (self.fc2_codes, self.fc2_scales)):
                mxfp4.check(mxfp4.Mxfp4(codes, scales), "Mxfp4Experts")
            self.shape1, self.shape2 = (mxfp4.Mxfp4(c, None).shape for c in (self.fc1_codes, self.fc2_codes))
        (e1, n1, h), (e2, h2, i) = self.shape1, self.shape2
        if e1 != e2 or n1 not in (i, 2 * i) or not e1 or h2 % 8 or self.base < 0:
            raise ValueError("Mxfp4Experts: fc1 [E, 2 I or I, H], fc2 [E, H_out, I], H_out a multiple of eight, base not negative")
        if e1 > MAX_EXPERTS:
            raise ValueError(f"Mxfp4Experts: {e1} experts, the kernels take {MAX_EXPERTS}")
        for tiled, codes, shape in ((self.tiled1, self.fc1_codes, self.shape1), (self.tiled2, self.fc2_codes, self.shape2)):
            if tiled is not None or codes is None:
                mxfp4.check_tiled(tiled, shape, "Mxfp4Experts")

    def __getstate__(self):
        """A copy or a pickle takes the tensors, not the structure of their addresses that `_struct` keeps here."""
        return {k: v for k, v in self.__dict__.items() if k != "_packed"}

    @property
    def experts(self) -> int:
        return self.shape1[0]

    @property
    def gated(self) -> bool:
        return self.shape1[1] == 2 * self.shape2[2]

    @property
    def bytes(self) -> int:
        (e, n1, h), (_, h2, i) = self.shape1, self.shape2
        return e * (n1 * h + h2 * i) * 17 // 32

    def held(self, fc1: bool) -> mxfp4.Mxfp4:
        """A stack's codes and scales by rows; from the kernels' layout where only that is left."""
        codes, scales = (self.fc1_codes, self.fc1_scales) if fc1 else (self.fc2_codes, self.fc2_scales)
        if codes is not None:
            return mxfp4.Mxfp4(codes, scales)
        return mxfp4.untile(self.tiled1 if fc1 else self.tiled2, *(self.shape1 if fc1 else self.shape2)[1:], gated=fc1 and self.gated)

    @classmethod
    def from_dense(cls, fc1: torch.Tensor, fc2: torch.Tensor, base: int = 0) -> "Mxfp4Experts":
        """Stacked BF16, FP16 or FP32 matrices, rounded to the format."""
        return cls(*mxfp4.quantize(fc1), *mxfp4.quantize(fc2), base=base)

    def __call__(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """`mxfp4_moe`, as a block that takes any experts calls it (`NemotronMoe`, its routed scaling factor in fc2 or the weights)."""
        return mxfp4_moe(self, x, ids, weights)


def tile(experts: Mxfp4Experts, release: bool = False) -> Mxfp4Experts:
    """Build the kernels' layout of both stacks (once); `release` drops the tensors by rows."""
    if experts.tiled1 is None:
        experts.tiled1 = mxfp4.tile(experts.held(True), gated=experts.gated)
    if experts.tiled2 is None:
        experts.tiled2 = mxfp4.tile(experts.held(False))
    if release:
        experts.fc1_codes = experts.fc1_scales = experts.fc2_codes = experts.fc2_scales = None
    return experts


def _struct(experts: Mxfp4Experts) -> _lib.HbMxfp4Experts:
    """The experts as the library takes them: built once, and again when a tensor or a number of `experts` was replaced."""
    if experts.tiled1 is None or experts.tiled2 is None:
        tile(experts)
    have = experts.__dict__.get("_packed")
    if have is None or have.of[0] is not experts.tiled1 or have.of[1] is not experts.tiled2 or have.of[2:] != (experts.base, experts.shape1, experts.shape2):
        (e, _, h), (_, h2, i) = experts.shape1, experts.shape2
        have = _lib.HbMxfp4Experts(experts.tiled1.data_ptr(), experts.tiled2.data_ptr(), e, experts.base, h, i, h2, int(experts.gated))
        have.of = (experts.tiled1, experts.tiled2, experts.base, experts.shape1, experts.shape2)
        have.at = C.byref(have)
        have.bytes_of = {}  # the workspace a call of (rows, k, pairs or a sum) takes
        experts._packed = have
    return have


def _ids32(ids: torch.Tensor) -> torch.Tensor:
    """Contiguous int32 ids. A wider one that int32 does not hold is outside of every range and stays so: cut off, it could name an expert."""
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, 2**31 - 1)
    return ids.to(torch.int32).contiguous()


def mxfp4_moe(experts: Mxfp4Experts, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, pairs: bool = False, pairs_bf16: bool = False) -> torch.Tensor:
    """Routed experts for x [M, H] BF16 with the router's ids [M, k] and weights [M, k] -> BF16 [M, H_out], the weighted sum of a row's pairs in
    FP32, added in an order that the sizes alone decide, and rounded once. An id outside this object's range base .. base + E - 1 adds nothing. With `pairs`, the FP32 (`pairs_bf16`:
    BF16) output of each (row, k) pair [M * k, H_out], unsummed and unweighted; rows of skipped pairs are unspecified."""
    if not isinstance(experts, Mxfp4Experts):
        raise ValueError("mxfp4_moe: on Mxfp4Experts")
    if x.dtype != torch.bfloat16 or x.ndim != 2 or x.shape[1] != experts.shape1[2]:
        raise ValueError("mxfp4_moe: x must be BF16 [M, hidden]")
    if ids.ndim != 2 or ids.shape[0] != x.shape[0] or weights.shape != ids.shape:
        raise ValueError("mxfp4_moe: ids and weights must be [M, k]")
    if ids.dtype not in ID_TYPES:
        raise ValueError("mxfp4_moe: ids must be whole numbers, int64 at most")
    st = _struct(experts)
    stream = _lib.stream_of(x, ids, weights, experts.tiled1, experts.tiled2)
    m, k = ids.shape
    mode = (2 if pairs_bf16 else 1) if pairs else 0
    out = x.new_empty((m * k if pairs else m, experts.shape2[1]), dtype=torch.float32 if mode == 1 else torch.bfloat16)
    if m == 0 or k == 0:
        return out if pairs else out.zero_()
    lib = _lib.lib()
    need = st.bytes_of.get((m, k, mode > 0))
    if need is None:
        if len(st.bytes_of) >= 4096:
            st.bytes_of.clear()
        need = st.bytes_of[m, k, mode > 0] = (lib.hb_mxfp4_moe_pairs_workspace_bytes if mode else lib.hb_mxfp4_moe_workspace_bytes)(st.at, m, k)
    ws = experts.tiled1.new_empty(max(need, 16))  # (of the capture's own pool in a captured call)
    # converted operands keep a name until the launches are enqueued
    ids32 = ids if ids.dtype == torch.int32 and ids.is_contiguous() else _ids32(ids)
    wt = weights if weights.dtype == torch.float32 and weights.is_contiguous() else weights.float().contiguous()
    xc = mxfp4.rows16(x)
    code = lib.hb_mxfp4_moe(st.at, xc.data_ptr(), ids32.data_ptr(), wt.data_ptr(), m, k, mode, out.data_ptr(), ws.data_ptr(), need, stream)
    if code:
        _lib.check(code, "mxfp4_moe")
    return out
