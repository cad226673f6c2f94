"""Low-rank adapters of many requests at once beside a shared projection, and their gradients: what a fine-tune learns around
frozen quantized weights, and what a server then holds beside them.

    out[r] = y[r] + scale_i (x[r] a_i^T) b_i,   i = index[r]

A pool holds the adapters of one projection [N, K], both matrices rank by rank: a [adapters, rank, K] and b [adapters, rank, N] (a
checkpoint's lora_B [N, rank], transposed once). So every product of the forward and the backward pass reads along a matrix's rows. Products
have FP32 sums; the sums between the two of an adapter keep all that FP32 holds of them (FP16: to 2^-37 of the largest), and the result is rounded
once. No counterpart in the reference.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

from hibana_amd import _lib
from hibana_amd.kernels.mxfp4 import TYPES

MOST, MOST_RANK = 4096, 256  # what the kernels take: adapters of a pool, their rank
INDEX = {torch.int32: 4, torch.int64: 8}


class Adapters:
    """a [adapters, rank, K] and b [adapters, rank, N] of one type (BF16, FP16 or FP32), contiguous. `scale`: FP32 [adapters] or a number (None: 1).
    `ranks` int32 [adapters]: how many of the `rank` rows are adapter i's (None: all; the rows behind them are not read). Tensors that require gradients get them through `add`."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | float | None = None, ranks: torch.Tensor | None = None):
        if isinstance(scale, (int, float)):
            scale = torch.full(a.shape[:1], float(scale), dtype=torch.float32, device=a.device)
        self._rooms: dict[tuple[int, int], int] = {}
        self.a, self.b, self.scale, self.ranks = a, b, scale, ranks
        self._check()

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        if name in ("a", "b", "scale", "ranks"):  # what the library was given last is not of these
            object.__setattr__(self, "_at", None)

    def _check(self) -> None:
        a, b, scale, ranks = self.a, self.b, self.scale, self.ranks
        if a.ndim != 3 or b.ndim != 3 or a.shape[:2] != b.shape[:2] or a.dtype != b.dtype or a.dtype not in TYPES or not a.numel() or not b.numel():
            raise ValueError("Adapters: a [adapters, rank, K] and b [adapters, rank, N], both BF16, FP16 or FP32")
        if a.shape[0] > MOST or a.shape[1] > MOST_RANK:
            raise ValueError(f"Adapters: up to {MOST} adapters of a rank up to {MOST_RANK}")
        if not a.is_contiguous() or not b.is_contiguous():
            raise ValueError("Adapters: a and b must be contiguous")
        if scale is not None and (scale.dtype != torch.float32 or scale.shape != a.shape[:1] or not scale.is_contiguous() or scale.requires_grad):
            raise ValueError("Adapters: scale FP32 [adapters], which takes no gradient")
        if ranks is not None and (ranks.dtype != torch.int32 or ranks.shape != a.shape[:1] or not ranks.is_contiguous()):
            raise ValueError("Adapters: ranks int32 [adapters]")
        if any(t is not None and t.device != a.device for t in (b, scale, ranks)):
            raise ValueError("Adapters: one device")

    @classmethod
    def from_pairs(cls, pairs, dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda") -> "Adapters":
        """A pool of the adapters (A [r, K], B [N, r], scale) as checkpoints hold them, of any ranks."""
        pairs = list(pairs)
        if not pairs or any(x.ndim != 2 or y.ndim != 2 or x.shape[0] != y.shape[1] or x.shape[1] != pairs[0][0].shape[1] or y.shape[0] != pairs[0][1].shape[0] for x, y, _ in pairs):
            raise ValueError("Adapters.from_pairs: (A [r, K], B [N, r], scale) of one projection")
        sizes = [x.shape[0] for x, _, _ in pairs]
        rank = max(max(sizes), 1)
        pool = cls(torch.zeros((len(pairs), rank, pairs[0][0].shape[1]), dtype=dtype, device=device), torch.zeros((len(pairs), rank, pairs[0][1].shape[0]), dtype=dtype, device=device),
                   torch.ones(len(pairs), dtype=torch.float32, device=device), torch.tensor(sizes, dtype=torch.int32, device=device))
        for i, pair in enumerate(pairs):
            pool.set(i, *pair)
        return pool

    def set(self, i: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Adapter i replaced by A [r, K], B [N, r], on the current stream. r below the pool's rank needs a pool with `ranks`, a scale one with `scale`."""
        n, rank, k = self.a.shape
        r = a.shape[0]
        if not 0 <= i < n or tuple(a.shape) != (r, k) or tuple(b.shape) != (self.out_features, r) or r > rank or (r < rank and self.ranks is None) or (scale != 1.0 and self.scale is None):
            raise ValueError(f"Adapters.set: an adapter A [r, {k}], B [{self.out_features}, r] of this pool (rank {rank}{'' if self.ranks is not None else ', all of them of it'})")
        with torch.no_grad():
            self.a[i, :r].copy_(a)
            self.b[i, :r].copy_(b.T)
            if self.scale is not None:
                self.scale[i].fill_(float(scale))
            if self.ranks is not None:
                self.ranks[i].fill_(r)

    @property
    def adapters(self) -> int:
        return self.a.shape[0]

    @property
    def rank(self) -> int:
        return self.a.shape[1]

    @property
    def in_features(self) -> int:
        return self.a.shape[2]

    @property
    def out_features(self) -> int:
        return self.b.shape[2]

    @property
    def bytes(self) -> int:
        return (self.a.numel() + self.b.numel()) * self.a.element_size()

    def __getstate__(self):
        """A copy or a pickle takes the tensors, not the structure of their addresses."""
        return {name: v for name, v in self.__dict__.items() if name not in ("_struct", "_at", "_rooms")}

    def __setstate__(self, state):
        self._rooms = {}
        for name, v in state.items():
            setattr(self, name, v)

    def struct(self):
        """What the library takes, looked at and made again where a tensor is another one, or its place, type or shape has changed (an optimizer may have put other memory
        in, at the old address too)."""
        a, b, scale, ranks = self.a, self.b, self.scale, self.ranks
        at = (a.data_ptr(), b.data_ptr(), None if scale is None else scale.data_ptr(), None if ranks is None else ranks.data_ptr(), a.shape, b.shape,
              a.dtype, b.dtype, a.is_contiguous(), b.is_contiguous(), scale is None or (scale.dtype, scale.numel(), scale.is_contiguous()),
              ranks is None or (ranks.dtype, ranks.numel(), ranks.is_contiguous()))
        if at != self._at:
            self._check()
            self._rooms.clear()
            n, rank, k = a.shape
            self._struct, self._at = C.byref(_lib.HbAdapters(*at[:4], n, rank, k, b.shape[2], TYPES[a.dtype])), at
        return self._struct

    def room(self, m: int, grads: int) -> int:
        need = self._rooms.get((m, grads))
        if need is None:
            if len(self._rooms) >= 4096:
                self._rooms.clear()
            need = _lib.lib().hb_adapters_workspace_bytes(self.struct(), m, grads)
            if not need:
                raise ValueError(f"adapters: up to 2^24 rows and axes of up to 2^22, not {m} rows beside a projection [{self.out_features}, {self.in_features}]")
            self._rooms[m, grads] = need
        return need


def _rows(t: torch.Tensor, width: int, pool: Adapters, what: str) -> torch.Tensor:
    if t.dtype != pool.a.dtype or t.ndim != 2 or t.shape[1] != width:
        raise ValueError(f"{what}: {pool.a.dtype} [M, {width}]")
    if t.is_contiguous():
        return t
    return t if t.stride(1) == 1 and (t.stride(0) >= width or t.shape[0] == 1) else t.contiguous()


def _stride(t: torch.Tensor, width: int) -> int:
    return width if t.is_contiguous() else max(t.stride(0), width)  # (that of a single row is nobody's)


def _operands(v: torch.Tensor, x: torch.Tensor, pool: Adapters, index: torch.Tensor, what: str):
    """The rows of v [M, N] and x [M, K] and the index as the library takes them, the number of rows and the current stream."""
    a = pool.a
    at = a.get_device()
    if v.ndim == 2 and v.is_contiguous() and x.is_contiguous() and index.is_contiguous() and v.dtype is a.dtype and x.dtype is a.dtype and index.dtype in INDEX \
            and v.get_device() == at and x.get_device() == at and index.get_device() == at and at >= 0 and at == torch._C._cuda_getDevice():
        m, n = v.shape
        if n == pool.b.shape[2] and x.shape == (m, a.shape[2]) and index.shape == (m,):  # as most calls are
            return v, x, index, m, torch._C._cuda_getCurrentRawStream(at)
    v, x = _rows(v, pool.b.shape[2], pool, what), _rows(x, a.shape[2], pool, what)
    m = v.shape[0]
    if x.shape[0] != m:
        raise ValueError(f"{what}: as many rows of x as there are results")
    if index.dtype not in INDEX or index.ndim != 1 or index.shape[0] != m:
        raise ValueError(f"{what}: an int32 or int64 index [{m}]")
    if not index.is_contiguous():
        index = index.contiguous()
    return v, x, index, m, _lib.stream_of(v, x, index, a)


def _add(y: torch.Tensor, x: torch.Tensor, pool: Adapters, index: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    yr, xr, ix, m, stream = _operands(y, x, pool, index, "adapters.add")
    k, n = pool.a.shape[2], pool.b.shape[2]
    if out is None:
        out = torch.empty_like(yr) if yr.is_contiguous() else yr.new_empty((m, n))
        to = n
    elif out.dtype != yr.dtype or out.shape != yr.shape or out.stride(1) != 1 or (m > 1 and out.stride(0) < n) or out.device != yr.device:
        raise ValueError("adapters.add: out like y, its rows contiguous")
    else:
        to = _stride(out, n)
    if m:
        struct = pool.struct()
        need = pool.room(m, 0)
        ws = yr.new_empty(need, dtype=torch.uint8)  # (of the capture's own pool in a captured call; a call's own, so that two at once share nothing)
        code = _lib.lib().hb_adapters_add(struct, xr.data_ptr(), _stride(xr, k), yr.data_ptr(), _stride(yr, n), ix.data_ptr(), INDEX[ix.dtype], m, out.data_ptr(), to,
                                          ws.data_ptr(), need, stream)
        if code:
            _lib.check(code, "adapters.add")
    return out


class _Add(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, scale, ranks, index, pool):
        ctx.save_for_backward(x, a, b, scale, ranks, index)  # (the pool may hold others when the gradient is asked for)
        return _add(y, x, pool, index, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, a, b, scale, ranks, index = ctx.saved_tensors
        _, need_x, need_a, need_b = ctx.needs_input_grad[:4]
        if not (need_x or need_a or need_b):
            return dy, *[None] * 7
        dx, da, db = grads(dy, x, Adapters(a.detach(), b.detach(), scale, ranks), index)
        return dy, dx if need_x else None, da.to(a.dtype) if need_a else None, db.to(b.dtype) if need_b else None, *[None] * 4


def add(y: torch.Tensor, x: torch.Tensor, pool: Adapters, index: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [M, N] plus each row's adapter of x [M, K], of the pool's type -> [M, N] (or `out`: y itself, or memory that no row of y has a part of: else refused). index int32 or int64 [M]: a row whose
    index is not of the pool (-1) is y's, bit for bit. Any order of rows: those of an adapter share one read of its matrices. An infinity in b (of the gradients: in a, x or
    dy) may come out as NaN: it is multiplied with values that are held in parts, some of them zero.

    Differentiable in y, x, pool.a and pool.b, in reverse (an input with a forward-mode tangent is refused). A training step that is to be captured calls `grads` itself: autograd's own streams and a
    capture do not go together, and the process would end; so a call that records a gradient is refused there. The framework's frozen linears
    record none of their rows: where x takes a gradient (adapters below this one), y has to as well, from a projection that gives dy W (a function
    of the program's own over `lin.dequantize()`; or y.requires_grad_(), whose gradient the program takes on itself); a y without one is refused."""
    if forward_ad._current_level >= 0:
        _lib.no_tangents("adapters.add", y, x, pool.a, pool.b, pool.scale)
    if torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or pool.a.requires_grad or pool.b.requires_grad or (out is not None and out.requires_grad)
                                    or (pool.scale is not None and pool.scale.requires_grad)):
        if out is not None:
            raise ValueError("adapters.add: no `out` where a gradient is recorded")
        if pool.scale is not None and pool.scale.requires_grad:
            raise ValueError("adapters.add: a pool's scale takes no gradient")
        if x.requires_grad and not y.requires_grad:
            raise ValueError("adapters.add: x takes a gradient and y none, so that the projection's own part of it, dy W, would be missing")
        if y.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("adapters.add: a captured step takes adapters.grads (no gradient is recorded in a capture)")
        return _Add.apply(y, x, pool.a, pool.b, pool.scale, pool.ranks, index, pool)
    got = _add(y, x, pool, index, out)
    if out is not None:
        torch._C._increment_version((out,))  # (`torch.autograd.graph.increment_version` at half its time)
    return got


def grads(dy: torch.Tensor, x: torch.Tensor, pool: Adapters, index: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of `add` given that of its result, dy [M, N]: (dx [M, K] of the pool's type, da FP32 [adapters, rank, K], db FP32 [adapters, rank,
    N]). An adapter that no row has gets zeros, as do the rows behind an adapter's rank; y's gradient is dy itself. Sums over rows are in a
    fixed order: the same call gives the same bits."""
    if forward_ad._current_level >= 0:
        _lib.no_tangents("adapters.grads", dy, x, pool.a, pool.b, pool.scale)
    dyr, xr, ix, m, stream = _operands(dy, x, pool, index, "adapters.grads")
    k, n = pool.a.shape[2], pool.b.shape[2]
    dx = xr.new_empty((m, k))
    if not m:
        return dx, torch.zeros(pool.a.shape, dtype=torch.float32, device=xr.device), torch.zeros(pool.b.shape, dtype=torch.float32, device=xr.device)
    da, db = xr.new_empty(pool.a.shape, dtype=torch.float32), xr.new_empty(pool.b.shape, dtype=torch.float32)
    struct = pool.struct()
    need = pool.room(m, 1)
    ws = xr.new_empty(need, dtype=torch.uint8)
    code = _lib.lib().hb_adapters_grads(struct, xr.data_ptr(), _stride(xr, k), dyr.data_ptr(), _stride(dyr, n), ix.data_ptr(), INDEX[ix.dtype], m, dx.data_ptr(), da.data_ptr(),
                                        db.data_ptr(), ws.data_ptr(), need, stream)
    if code:
        _lib.check(code, "adapters.grads")
    return dx, da, db
