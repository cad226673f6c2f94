"""Kernel entry points of the quantized linear / MoE path (hibana/kernels/ops.py:50-92 of the reference, plus the
routing and combine ops of hibana/kernels/flashnext_fused.py that sit either side of the experts)."""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from hibana_amd import _lib
from hibana_amd.kernels import adapters, mxfp4, w3
from hibana_amd.weights.mxfp4 import Mxfp4Linear


def w3_decode(lin, m: int, rows: int | None = None) -> bool:
    """True when this call runs the 3-bit decode copy instead of the NVFP4 weights: at most `rows` rows (None:
    w3.MAX_ROWS) (hibana/kernels/ops.py:50-53)."""
    return lin.w3 is not None and m <= (rows or w3.MAX_ROWS) and w3.enabled()


def nvfp4_linear(x: torch.Tensor, lin, prequantized=None, relu2: bool = False) -> torch.Tensor:
    """BF16 x [M, K] -> BF16 [M, N] on NVFP4 weights, weight-only: bf16((x Wq^T)_fp32 * global scale); the 3-bit copy
    serves the call when one is attached and enabled (hibana/kernels/ops.py:56-83). No host synchronization on the
    call path once `lin.tile()` has run (it caches the global scale as a host float), so the call can be captured."""
    if prequantized is not None:
        raise ValueError("nvfp4_linear: NVFP4 activations are not taken by the weight-only kernels")
    if x.dtype == torch.bfloat16 and w3_decode(lin, x.shape[0]) and not relu2:
        return w3.w3_linear(x, lin.w3)
    if x.dtype != torch.bfloat16 or x.ndim != 2 or x.shape[1] != lin.in_features:
        raise ValueError("nvfp4_linear: x must be BF16 [M, in_features]")
    _lib.need_gpu(x)
    if lin.tiled is None or lin.scale2 is None:
        lin.tile()
    m, n, k = x.shape[0], lin.out_features, lin.in_features
    y = x.new_empty((m, n))
    if m:
        lib = _lib.lib()
        xc = x.contiguous()  # held until the launch is enqueued: a temporary's block could be handed out again before that
        need = lib.hb_nvfp4_gemm_room_bytes(m, n, k) if m > 16 else 0  # where K is shared among workgroups
        ws = _lib.workspace(x.device, need, "gemm") if need else None
        code = lib.hb_nvfp4_gemm_ws(xc.data_ptr(), m, lin.tiled.data_ptr(), lin.scale2, n, k, int(relu2), y.data_ptr(), _lib.ptr(ws), need, _lib.stream())
        if code:
            _lib.check(code, "nvfp4_linear")
    return y


def mxfp4_linear(x, lin, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x [M, K] -> [M, N] on a `Mxfp4Linear`: both operands in the microscaled four-bit format, FP32 sums rounded once. x is BF16,
    FP16 or FP32, rounded to the format on the way (`mxfp4.quantize`'s codes), and the result of its type; or a `mxfp4.Mxfp4` that
    holds it already, and the result of `dtype`. Once `lin.tile()` has run the call can be captured."""
    ready = isinstance(x, mxfp4.Mxfp4)
    kind = mxfp4.CODES if ready else mxfp4.TYPES.get(x.dtype)
    out_type = dtype if ready else x.dtype
    to = mxfp4.TYPES.get(out_type)
    if type(lin) is not Mxfp4Linear and not isinstance(lin, Mxfp4Linear):  # (the layout of another format is not told from this one's)
        raise ValueError("mxfp4_linear: on an Mxfp4Linear")
    if kind is None or to is None or len(x.shape) != 2 or x.shape[1] != lin.in_features:
        raise ValueError("mxfp4_linear: x must be BF16, FP16 or FP32 [M, in_features], or hold such rows")
    if lin.tiled is None:
        lin.tile()
    if ready:
        at, scales, held, stream = mxfp4.places(x, "mxfp4_linear")
        _lib.need_one_gpu(lin.tiled)
    else:
        stream = _lib.stream_of(x, lin.tiled)
        held = mxfp4.rows16(x)  # held until the launch is enqueued
        at, scales = held.data_ptr(), None
    m, n, k = x.shape[0], lin.out_features, lin.in_features
    y = lin.tiled.new_empty((m, n), dtype=out_type)
    if m:
        lib = _lib.lib()
        need = lin.rooms.get((m, kind))
        if need is None:
            if len(lin.rooms) >= 4096:
                lin.rooms.clear()
            need = lin.rooms[m, kind] = lib.hb_mxfp4_linear_workspace_bytes(m, n, k, kind)
        ws = lin.tiled.new_empty(need) if need else None  # (of the capture's own pool in a captured call)
        code = lib.hb_mxfp4_linear(at, scales, kind, m, lin.tiled.data_ptr(), n, k, y.data_ptr(), to, _lib.ptr(ws), need, stream)
        if code:
            _lib.check(code, "mxfp4_linear")
    return y


def silu_and_mul(gate_up: torch.Tensor, pairs: int = 0) -> torch.Tensor:
    """silu(gate) * up of BF16 [..., gate | up], or (`pairs`) of gate and up alternating in blocks of `pairs` columns
    (hibana/kernels/ops.py:86-92), on the GPU; the roundings are those of the BF16 tensor expression."""
    if gate_up.dtype != torch.bfloat16 or gate_up.shape[-1] % 4 or (pairs and (pairs % 2 or (gate_up.shape[-1] // 2) % pairs)):
        raise ValueError("silu_and_mul: BF16 [..., 2 * half], half even (and a multiple of an even `pairs`)")
    _lib.need_gpu(gate_up)
    half = gate_up.shape[-1] // 2
    flat = (gate_up if gate_up.ndim == 2 else gate_up.reshape(-1, 2 * half)).contiguous()
    out = flat.new_empty((flat.shape[0], half))
    if flat.shape[0]:
        code = _lib.lib().hb_silu_and_mul(flat.data_ptr(), flat.shape[0], half, pairs, out.data_ptr(), _lib.stream())
        if code:
            _lib.check(code, "silu_and_mul")
    return out if gate_up.ndim == 2 else out.reshape(*gate_up.shape[:-1], half)


def silu_mul(gate_up: torch.Tensor, pairs: int = 0) -> torch.Tensor:
    """bf16(silu(gate) * up) of BF16 [M, 2 I] from the FP32 product, one rounding (hibana/kernels/flashnext_fused.py:
    624-639); columns as in `silu_and_mul`."""
    if gate_up.dtype != torch.bfloat16 or gate_up.ndim != 2 or gate_up.shape[1] % 4:
        raise ValueError("silu_mul: BF16 [M, 2 I] with I even")
    half = gate_up.shape[1] // 2
    if pairs and (pairs % 2 or half % pairs):
        raise ValueError("silu_mul: pairs must be even and divide I")
    _lib.need_gpu(gate_up)
    gu = gate_up.contiguous()
    out = torch.empty((gu.shape[0], half), dtype=torch.bfloat16, device=gu.device)
    if gu.shape[0]:
        _lib.check(_lib.lib().hb_silu_mul(_lib.ptr(gu), gu.shape[0], half, pairs, _lib.ptr(out), _lib.stream()), "silu_mul")
    return out


def silu_mul_quant_groups(gate_up: torch.Tensor, pairs: int = 0, torch_chain: bool = False):
    """`w3.quant_groups(silu_mul(gate_up))` in one launch, bit for bit: BF16 [M, 2I] -> (E4M3 [M, I], FP32 scales
    [M, I/32]); `pairs`: gate and up interleaved in blocks of that many columns; `torch_chain`: the product as
    `silu_and_mul` rounds it (hibana/kernels/flashnext_fused.py:841-853), the dense MLP's 3-bit decode input
    (hibana/model/mlp.py:36-42)."""
    if gate_up.dtype != torch.bfloat16 or gate_up.ndim != 2 or gate_up.stride(1) != 1 or gate_up.shape[1] % 64:
        raise ValueError("silu_mul_quant_groups: BF16 [M, 2 I] with I a multiple of 32")
    half = gate_up.shape[1] // 2
    if pairs and (pairs % 32 or half % pairs):
        raise ValueError("silu_mul_quant_groups: pairs must be a multiple of 32 dividing I")
    _lib.need_gpu(gate_up)
    gu = gate_up.contiguous()
    m = gu.shape[0]
    q = gu.new_empty((m, half), dtype=torch.float8_e4m3fn)
    scales = gu.new_empty((m, half // 32), dtype=torch.float32)
    if m:
        code = _lib.lib().hb_silu_mul_quant_groups(gu.data_ptr(), m, half, pairs, int(torch_chain), q.data_ptr(), scales.data_ptr(), _lib.stream())
        if code:
            _lib.check(code, "silu_mul_quant_groups")
    return q, scales


def silu_mul_quant_mxfp4(gate_up: torch.Tensor, pairs: int = 0) -> mxfp4.Mxfp4:
    """silu(gate) * up of [..., 2 I] (BF16, FP16 or FP32) rounded to the microscaled four-bit format in the same launch: the codes
    that the product in 64 bits has; columns gate | up, or (`pairs`, a multiple of eight) both alternating in blocks of that many. I a
    multiple of 32. A group with an infinite or undefined product stands for NaN."""
    kind = mxfp4.TYPES.get(gate_up.dtype)
    if kind is None or gate_up.ndim == 0 or gate_up.shape[-1] % 64:
        raise ValueError("silu_mul_quant_mxfp4: BF16, FP16 or FP32 [..., 2 I] with I a multiple of 32")
    half = gate_up.shape[-1] // 2
    if pairs and (pairs < 0 or pairs % 8 or half % pairs):
        raise ValueError("silu_mul_quant_mxfp4: pairs must be a multiple of eight dividing I")
    stream = _lib.stream_of(gate_up)
    n = gate_up.numel() // 2
    block = gate_up.new_empty(n // mxfp4.GROUP * 17, dtype=torch.uint8)
    if n:
        gu = mxfp4.rows16(gate_up)  # held until the launch is enqueued
        at = block.data_ptr()
        code = _lib.lib().hb_silu_mul_quant_mxfp4(gu.data_ptr(), kind, n // half, half, pairs, at, at + n // 2, stream)
        if code:
            _lib.check(code, "silu_mul_quant_mxfp4")
    return mxfp4.Mxfp4.of_block(block, (*gate_up.shape[:-1], half))


def route_topk(logits: torch.Tensor, k: int, slots: torch.Tensor | None = None, steps: int = 1, repeat: bool = False):
    """[M, E] FP32 logits -> (int32 ids [M, k], FP32 renormalized softmax weights [M, k]), largest first. With `slots`,
    row r is real iff slots[r // steps] != 0; a padded row takes expert E at weight 0 (the 3-bit experts skip it) or,
    `repeat`, row 0's first choice at weight 0 (hibana/kernels/flashnext_fused.py:308-319)."""
    _lib.need_gpu(logits, slots)
    m, e = logits.shape
    lg = logits.float().contiguous()
    sl = None if slots is None else slots.to(torch.int32).contiguous()
    ids = torch.empty((m, k), dtype=torch.int32, device=logits.device)
    w = torch.empty((m, k), dtype=torch.float32, device=logits.device)
    if m:
        _lib.check(_lib.lib().hb_route_softmax_topk(_lib.ptr(lg), m, e, k, _lib.ptr(sl), steps, int(repeat), _lib.ptr(ids), _lib.ptr(w),
                                                    _lib.stream()), "route_topk")
    return ids, w


SCORING = {"softmax": 0, "sigmoid": 1}  # HB_SOFTMAX, HB_SIGMOID


@dataclass(frozen=True, eq=False)
class Routing:
    """How `route_experts` routes, for a layer that holds it (`MoeLayer(routing=...)`)."""
    scoring: str = "softmax"
    bias: torch.Tensor | None = None  # FP32 [E]
    groups: int = 1
    kept: int = 1
    renormalize: bool = True
    scale: float = 1.0

    def __call__(self, logits: torch.Tensor, k: int, slots: torch.Tensor | None = None, steps: int = 1):
        return route_experts(logits, k, self.scoring, bias=self.bias, groups=self.groups, kept=self.kept, renormalize=self.renormalize, scale=self.scale, slots=slots, steps=steps)


def _route_logits(logits: torch.Tensor, scoring: str, what: str) -> torch.Tensor:
    if logits.dtype not in mxfp4.TYPES or logits.ndim != 2 or scoring not in SCORING or logits.shape[0] > 1 << 25:
        raise ValueError(f"{what}: BF16, FP16 or FP32 logits [M, E] of up to 2^25 rows, scoring softmax or sigmoid")
    return logits if logits.is_contiguous() or (logits.stride(1) == 1 and logits.stride(0) >= logits.shape[1]) else logits.contiguous()


def _route_experts(logits: torch.Tensor, k: int, scoring: str, bias, groups: int, kept: int, renormalize: bool, scale: float, slots, steps: int):
    what = "route_experts"
    lg = _route_logits(logits, scoring, what)
    m, e = lg.shape
    if not (1 <= e <= 1024 and 1 <= kept <= groups <= 64 and e % groups == 0 and 1 <= k <= min(63, kept * (e // groups))):
        raise ValueError(f"{what}: up to 1024 experts in up to 64 groups of a size, k up to 63 and the experts of the kept groups")
    lanes = 1 << (64 // groups).bit_length() - 1  # of a wavefront that a group has, up to sixteen experts in each
    if e // groups > 16 * lanes:
        raise ValueError(f"{what}: {groups} groups have up to {16 * lanes} experts each")
    bias32 = sl = None
    if bias is not None:
        if bias.ndim != 1 or bias.shape[0] != e or not bias.is_floating_point():
            raise ValueError(f"{what}: a bias [E]")
        bias32 = bias if bias.dtype == torch.float32 and bias.is_contiguous() else bias.float().contiguous()
    if steps < 1 or m % steps or (slots is not None and slots.numel() < m // steps):
        raise ValueError(f"{what}: whole requests of `steps` rows, a slot for every request")
    if slots is not None:
        sl = slots if slots.dtype == torch.int32 and slots.is_contiguous() else slots.ne(0).to(torch.int32).contiguous()  # (what 32 bits do not hold stays apart from 0)
    stream = _lib.stream_of(lg, *(t for t in (bias32, sl) if t is not None))
    ids, weights = lg.new_empty((m, k), dtype=torch.int32), lg.new_empty((m, k), dtype=torch.float32)
    if m:
        code = _lib.lib().hb_route_experts(lg.data_ptr(), mxfp4.TYPES[lg.dtype], max(lg.stride(0), e), m, e, k, SCORING[scoring], _lib.ptr(bias32), groups, kept, int(renormalize),
                                           scale, _lib.ptr(sl), steps, ids.data_ptr(), weights.data_ptr(), stream)
        if code:
            _lib.check(code, what)
    return ids, weights


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, scoring, renormalize, scale, *rest):
        bias, groups, kept, slots, steps = rest
        ids, weights = _route_experts(logits, k, scoring, bias, groups, kept, renormalize, scale, slots, steps)
        ctx.save_for_backward(logits, ids)
        ctx.rule = scoring, renormalize, scale
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, dweights):
        logits, ids = ctx.saved_tensors
        scoring, renormalize, scale = ctx.rule
        return (route_experts_grad(dweights, logits, ids, scoring, renormalize=renormalize, scale=scale), *[None] * 9)


def route_experts(logits: torch.Tensor, k: int, scoring: str = "softmax", *, bias: torch.Tensor | None = None, groups: int = 1, kept: int = 1, renormalize: bool = True,
                  scale: float = 1.0, slots: torch.Tensor | None = None, steps: int = 1):
    """logits [M, E] (BF16, FP16 or FP32; E up to 1024) -> (int32 ids [M, k], FP32 weights [M, k]), largest choice first. Scores are the logits' softmax or
    sigmoid; the choice goes by score + bias (FP32 [E], None: 0) among the experts of the `kept` groups (of `groups`, of consecutive experts, up to 16 times the power of
    two that 64 / groups holds: all that there are where the groups are a power of two) whose best two sum highest; equal ones by the lower number. Without a bias the order is the logits' own, else (and between groups) that of the values in FP64. Weights are the plain scores, with
    `renormalize` divided by their sum, times `scale`. An expert whose logit is -inf (a mask) or NaN is never chosen: slots left over, and all of a padded row's
    (slots[r // steps] == 0), have id E, which the experts' kernels skip, and weight 0. A row that has a NaN logit has NaN weights.

    Differentiable in the logits, in reverse (a forward-mode tangent is refused), through the weights (the bias only moves the choice). A captured training step calls `route_experts_grad`
    itself: a call that records a gradient is refused in a capture, as in `adapters.add`. The experts' calls read the weights' values alone and record
    nothing: a router that learns sums their pairs (`pairs=True`) with the weights itself. No counterpart in the reference."""
    if forward_ad._current_level >= 0:
        _lib.no_tangents("route_experts", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        if logits.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("route_experts: a captured step takes route_experts_grad (no gradient is recorded in a capture)")
        return _RouteExperts.apply(logits, k, scoring, renormalize, scale, bias, groups, kept, slots, steps)
    return _route_experts(logits, k, scoring, bias, groups, kept, renormalize, scale, slots, steps)


def route_experts_grad(dweights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, scoring: str = "softmax", *, renormalize: bool = True,
                       scale: float = 1.0) -> torch.Tensor:
    """The gradient of `route_experts`' logits [M, E], of their type, given that of its weights (FP32 [M, k]) and the ids it chose (int32 [M, k]; one
    outside 0 .. E - 1 adds nothing)."""
    what = "route_experts_grad"
    if forward_ad._current_level >= 0:
        _lib.no_tangents(what, dweights, logits)
    lg = _route_logits(logits, scoring, what)
    m, e = lg.shape
    if ids.dtype != torch.int32 or ids.ndim != 2 or ids.shape[0] != m or dweights.dtype != torch.float32 or dweights.shape != ids.shape:
        raise ValueError(f"{what}: dweights FP32 and ids int32, both [M, k]")
    dw, chosen = dweights.contiguous(), ids.contiguous()
    stream = _lib.stream_of(lg, dw, chosen)
    out = lg.new_empty((m, e))
    if m:
        code = _lib.lib().hb_route_experts_grad(dw.data_ptr(), lg.data_ptr(), mxfp4.TYPES[lg.dtype], max(lg.stride(0), e), chosen.data_ptr(), m, e, chosen.shape[1],
                                                SCORING[scoring], int(renormalize), scale, out.data_ptr(), stream)
        if code:
            _lib.check(code, what)
    return out


def adapted_linear(x: torch.Tensor, lin, pool: adapters.Adapters, index: torch.Tensor) -> torch.Tensor:
    """A linear's rows (any of the `Linear` protocol: three-bit, NVFP4 or MXFP4 weights) with each row's own adapter of `pool` beside it
    (`adapters.add` into the linear's fresh result): the serving form, without gradients."""
    if pool.in_features != lin.in_features or pool.out_features != lin.out_features:
        raise ValueError(f"adapted_linear: adapters of a projection [{pool.out_features}, {pool.in_features}] beside one [{lin.out_features}, {lin.in_features}]")
    y = lin(x)
    with torch.no_grad():
        return adapters.add(y, x, pool, index, out=y)


ROUTE_CANDIDATES = 20  # a row takes its experts from its 20 largest logits


def route_budget(logits: torch.Tensor, k: int, keep: int, budget: int, slots: torch.Tensor | None = None, steps: int = 1,
                 repeat: bool = False, per_request: int = 0, min_cap: int = 0):
    """Budgeted top-k (hibana/kernels/flashnext_fused.py:462-502): BF16 [R, E] logits -> (int32 ids [R, k], FP32 weights
    [R, k]). The experts the call reads are chosen for the whole call under a cap: every real row's top `keep`, then the
    experts with the most softmax probability within the real rows' top k until the set holds the cap (`budget`, or
    with `per_request`, min(budget, max(min_cap, per_request x the real requests))); each real row takes its candidates
    (its 20 largest logits, an exact tie to the lower expert) in the set, in rank order, up to k, its weights the
    softmax over E renormalized over them. Slots left over (all of a padded row's: slots[r // steps] == 0) hold id E at
    weight 0, or with `repeat` the row's top 1 (a padded row: row 0's)."""
    if logits.dtype != torch.bfloat16 or logits.ndim != 2:
        raise ValueError("route_budget: BF16 [R, E] logits")
    r, e = logits.shape
    if not (ROUTE_CANDIDATES <= e <= 1024 and 1 <= k <= ROUTE_CANDIDATES and 0 <= keep <= ROUTE_CANDIDATES) or budget < 0 or steps < 1 or r % steps:
        raise ValueError("route_budget: 20 <= E <= 1024, k and keep at most 20, whole requests of `steps` rows")
    if slots is not None and slots.numel() < r // steps:
        raise ValueError("route_budget: a slot for every request")
    _lib.need_gpu(logits, slots)
    lg = logits.contiguous()
    sl = None if slots is None else slots.to(torch.int32).contiguous()
    ids = torch.empty((r, k), dtype=torch.int32, device=logits.device)
    w = torch.empty((r, k), dtype=torch.float32, device=logits.device)
    if r:
        ws = torch.empty((_lib.lib().hb_route_budget_workspace_bytes(r),), dtype=torch.uint8, device=logits.device)
        _lib.check(_lib.lib().hb_route_budget(_lib.ptr(lg), r, e, k, keep, budget, _lib.ptr(sl), steps, int(repeat), per_request, min_cap,
                                              _lib.ptr(ws), ws.numel(), _lib.ptr(ids), _lib.ptr(w), _lib.stream()), "route_budget")
    return ids, w


def moe_combine_pairs(y: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, shared: torch.Tensor | None, x: torch.Tensor | None,
                      gate_w: torch.Tensor | None, e_lo: int = 0, e_n: int = 512) -> torch.Tensor:
    """bf16(bf16(sum_k w_k y_k over this rank's pairs, in slot order) + sigmoid(x . gate_w) * shared) from the unsummed
    pair outputs y [m * topk, H] (FP32 or BF16) (hibana/kernels/flashnext_fused.py:556-571). `shared` None: the
    routed sum alone; `gate_w` None: the shared output is added ungated."""
    _lib.need_gpu(y, ids, weights)
    m, topk = ids.shape
    h = y.shape[1]
    out = torch.empty((m, h), dtype=torch.bfloat16, device=y.device)
    if m == 0:
        return out
    if y.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("moe_combine_pairs: pairs must be FP32 or BF16")
    if y.shape[0] != m * topk or weights.shape != ids.shape or (shared is not None and tuple(shared.shape) != (m, h)):
        raise ValueError("moe_combine_pairs: y [M * k, H], ids / weights [M, k], shared [M, H]")
    if gate_w is not None and shared is not None and (x is None or tuple(x.shape) != (m, h) or gate_w.numel() != h):
        raise ValueError("moe_combine_pairs: the gate takes x [M, H] and gate_w [H] (the layer's input rows)")
    # every converted operand is bound to a name until the launch is enqueued
    yc, ids32, wt = y.contiguous(), ids.to(torch.int32).contiguous(), weights.float().contiguous()
    sh = None if shared is None else shared.to(torch.bfloat16).contiguous()
    xx = None if x is None else x.to(torch.bfloat16).contiguous()
    gw = None if gate_w is None else gate_w.float().reshape(-1).contiguous()
    _lib.check(_lib.lib().hb_moe_combine_pairs(_lib.ptr(yc), int(y.dtype == torch.bfloat16), _lib.ptr(ids32), _lib.ptr(wt), _lib.ptr(sh),
                                               _lib.ptr(xx), _lib.ptr(gw), e_lo, e_n, m, topk, h, _lib.ptr(out), _lib.stream()),
               "moe_combine_pairs")
    return out


def moe_combine(routed: torch.Tensor, shared: torch.Tensor, x: torch.Tensor, gate_w: torch.Tensor) -> torch.Tensor:
    """bf16(routed + sigmoid(x . gate_w) * shared) for BF16 routed / shared [M, H] (hibana/kernels/flashnext_fused.py:
    506-526): the combine kernel on one pair a row at weight 1, whose rounded sum is `routed` itself."""
    if routed.dtype != torch.bfloat16 or routed.ndim != 2 or shared.shape != routed.shape or x.shape != routed.shape or gate_w.numel() != routed.shape[1]:
        raise ValueError("moe_combine: routed, shared and x must be BF16 [M, H] of one shape, gate_w [H]")
    m = routed.shape[0]
    ids = torch.zeros((m, 1), dtype=torch.int32, device=routed.device)
    ones = torch.ones((m, 1), dtype=torch.float32, device=routed.device)
    return moe_combine_pairs(routed, ids, ones, shared, x, gate_w, 0, 1)

