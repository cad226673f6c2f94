"""What learns around frozen quantized weights, as a server and a training step call it: low-rank adapters beside a shared
projection, many requests' at once, with their gradients, and the routing of rows to experts, with its gradient.

Every case is a dict of plain values whose "path" names the operator:

  add         out = y + scale_i (x a_i^T) b_i for every row's own adapter i: x [rows, in], y [rows, out], a [adapters, rank, in],
              b [adapters, rank, out], all of "dtype". "runs": 0: every row a request of its own (decode), else the rows of that
              many sequences one behind the other; "ragged": the adapters have ranks of their own, up to "rank" (the rows of a
              and b behind them are not the adapter's); "none": that many requests (rows, or sequences) have no adapter
  grads       of the same, given dy [rows, out]: dx (of "dtype"), da and db (in 32 bits, zero where no row has the adapter)
  route       logits [rows, experts] of "dtype" -> each row's topk experts and their weights: scores are the softmax or the sigmoid
              of the logits, the choice goes by score + bias, among the experts of the "kept" groups (of "groups") whose best
              two sum highest; weights are the plain scores, divided by their sum with "renorm", times "scale". An expert
              whose logit is -inf is never chosen; slots left over, and all of the "padded" last rows', name no expert
              (id = experts, weight 0). "masked": the share of the logits that are -inf (and all of the first row's)
  route_grad  the gradient of the logits, given that of the weights
"""
from __future__ import annotations

import functools
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_FLOPS = 2.2e10  # of a drawn case: below the largest listed one's
MOST_BYTES = 4.8e8


def listed() -> list[dict]:
    return [
        # one decoded token through an attention-sized projection: the smallest call
        {"name": "add_1", "path": "add", "rows": 1, "in": 5120, "out": 5120, "rank": 16, "adapters": 8, "runs": 0, "ragged": False, "none": 0, "dtype": "bf16"},
        # a decode batch of many requests beside an MLP's up projection, adapters of different ranks, some requests without
        {"name": "add_64", "path": "add", "rows": 64, "in": 5120, "out": 25600, "rank": 64, "adapters": 32, "runs": 0, "ragged": True, "none": 8, "dtype": "bf16"},
        # a verify batch of five requests in fp16 beside a projection of odd width
        {"name": "add_f16_77", "path": "add", "rows": 77, "in": 5120, "out": 2049, "rank": 24, "adapters": 16, "runs": 5, "ragged": False, "none": 0, "dtype": "f16"},
        # a prefill batch of eight sequences, one of them without an adapter
        {"name": "add_4096", "path": "add", "rows": 4096, "in": 5120, "out": 5120, "rank": 32, "adapters": 6, "runs": 8, "ragged": False, "none": 1, "dtype": "bf16"},
        # a small training step in 32 bits on odd sizes
        {"name": "grads_f32_333", "path": "grads", "rows": 333, "in": 1000, "out": 2049, "rank": 12, "adapters": 3, "runs": 7, "ragged": False, "none": 0, "dtype": "f32"},
        # a training step of one adapter; of four tasks together, down an MLP's projection (the most work)
        {"name": "grads_2048", "path": "grads", "rows": 2048, "in": 5120, "out": 5120, "rank": 16, "adapters": 1, "runs": 1, "ragged": False, "none": 0, "dtype": "bf16"},
        {"name": "grads_f16_8192", "path": "grads", "rows": 8192, "in": 12800, "out": 2560, "rank": 64, "adapters": 4, "runs": 16, "ragged": True, "none": 0, "dtype": "f16"},
        # one token's routing; a prefill chunk's among groups, by sigmoid scores and a bias for balance; a ragged batch with
        # experts masked out and padded rows
        {"name": "route_1", "path": "route", "rows": 1, "experts": 512, "topk": 10, "scoring": "softmax", "bias": False, "groups": 1, "kept": 1, "renorm": True, "scale": 1.0,
         "masked": 0.0, "padded": 0, "dtype": "bf16"},
        {"name": "route_8192", "path": "route", "rows": 8192, "experts": 256, "topk": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "kept": 4, "renorm": True, "scale": 2.5,
         "masked": 0.0, "padded": 0, "dtype": "f32"},
        {"name": "route_f16_777", "path": "route", "rows": 777, "experts": 60, "topk": 4, "scoring": "softmax", "bias": True, "groups": 1, "kept": 1, "renorm": False, "scale": 1.0,
         "masked": 0.1, "padded": 9, "dtype": "f16"},
        # the routers' gradients in a training step: of all the scores through the softmax's sum; of the chosen ones alone
        {"name": "route_grad_2049", "path": "route_grad", "rows": 2049, "experts": 512, "topk": 10, "scoring": "softmax", "bias": False, "groups": 1, "kept": 1, "renorm": False,
         "scale": 1.0, "masked": 0.0, "padded": 0, "dtype": "bf16"},
        {"name": "route_grad_8192", "path": "route_grad", "rows": 8192, "experts": 256, "topk": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "kept": 4, "renorm": True,
         "scale": 2.5, "masked": 0.0, "padded": 0, "dtype": "f32"},
    ]


def _between(rng, low: float, high: float) -> int:
    """A whole number between the two, spread evenly over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    path = rng.choice(["add", "add", "add", "grads", "grads", "route", "route", "route_grad"])
    if path in ("add", "grads"):
        case = {"path": path, "rows": _between(rng, 1, 4096) if path == "add" else _between(rng, 16, 8192), "in": _between(rng, 64, 12800), "out": _between(rng, 64, 25600),
                "rank": _between(rng, 1, 128), "adapters": _between(rng, 1, 48 if path == "add" else 8)}
        case["runs"] = min(case["rows"], _between(rng, 1, 24))
        if path == "add" and case["rows"] <= 256 and rng.random() < 0.6:
            case["runs"] = 0
        requests = case["runs"] or case["rows"]
        case |= {"ragged": rng.random() < 0.4, "none": rng.choice([0, 0, requests // 5]), "dtype": rng.choice(list(TYPES))}
        while work(case)["flops"] > MOST_FLOPS or work(case)["bytes"] > MOST_BYTES:
            case["rows"] = max(requests, case["rows"] * 3 // 4)
            case["out"] = max(64, case["out"] * 7 // 8)
            case["in"] = max(64, case["in"] * 7 // 8)
        return case
    groups = rng.choice([1, 1, 2, 4, 8, 16])
    experts = groups * _between(rng, max(2, 8 // groups), 1024 // groups)
    kept = rng.randint((groups + 1) // 2, groups)
    rows = _between(rng, 1, 16384)
    return {"path": path, "rows": rows, "experts": experts, "topk": rng.randint(1, min(22, kept * (experts // groups))), "scoring": rng.choice(["softmax", "sigmoid"]),
            "bias": rng.random() < 0.5, "groups": groups, "kept": kept, "renorm": rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]),
            "masked": rng.choice([0.0, 0.0, 0.2]), "padded": rng.choice([0, 0, rows // 6]), "dtype": rng.choice(list(TYPES))}


# ------------------------------------------------------------------------------------------------ the plain form

def _columns(s: SimpleNamespace):
    """(a [adapters * rank, in], b [adapters * rank, out], FP32 [rows, adapters * rank]: a row's scale in the columns of its own
    adapter, zero in the others'): the sum over all the columns is then that of the row's own."""
    n, rank, _ = s.a.shape
    mine = s.index[:, None] == torch.arange(n, device=s.index.device)[None, :]
    used = torch.arange(rank, device=s.index.device)[None, :] < s.ranks[:, None]
    factor = torch.where(mine, s.scale[None, :], 0.0)[:, :, None] * used[None, :, :]
    return s.a.float().flatten(0, 1), s.b.float().flatten(0, 1), factor.flatten(1)


def _plain_add(s: SimpleNamespace) -> torch.Tensor:
    a, b, factor = _columns(s)
    return (s.y.float() + (s.x.float() @ a.T * factor) @ b).to(s.y.dtype)


def _plain_grads(s: SimpleNamespace):
    a, b, factor = _columns(s)
    x, dy = s.x.float(), s.dy.float()
    inner = dy @ b.T * factor
    da = inner.T @ x
    db = (x @ a.T * factor).T @ dy
    return (inner @ a).to(s.x.dtype), da.unflatten(0, s.a.shape[:2]), db.unflatten(0, s.b.shape[:2])


def _scores(logits: torch.Tensor, scoring: str) -> torch.Tensor:
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(e.dtype).tiny)


def _plain_route(s: SimpleNamespace):
    rows, experts = s.logits.shape
    logits = s.logits.double()  # 64 bits: which of two near choices is the larger
    score = _scores(logits, s.scoring)
    choice = score if s.bias is None else score + s.bias.double()
    choice = choice.masked_fill(torch.isneginf(logits), -math.inf)
    if s.groups > 1:
        best = choice.unflatten(1, (s.groups, -1)).sort(-1, descending=True).values
        best = best[..., 0] + (0.0 if best.shape[-1] == 1 else torch.where(torch.isneginf(best[..., 1]), 0.0, best[..., 1]))
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :s.kept]
        open_ = torch.zeros(rows, s.groups, dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        choice = choice.masked_fill(~open_.repeat_interleave(experts // s.groups, 1), -math.inf)
    top, ids = (t[:, :s.topk] for t in choice.sort(dim=-1, descending=True, stable=True))
    real = ~torch.isneginf(top)
    if s.slots is not None:
        real &= s.slots[:, None] != 0
    weights = torch.where(real, torch.gather(score, 1, ids), 0.0)
    if s.renorm:
        weights = weights / weights.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float64).tiny)
    return torch.where(real, ids, experts).to(torch.int32), (weights * s.scale).float()


def _plain_route_grad(s: SimpleNamespace) -> torch.Tensor:
    rows, experts = s.logits.shape
    score = _scores(s.logits.float(), s.scoring)
    real = s.ids < experts
    at = torch.where(real, s.ids, 0).long()
    mine = torch.where(real, torch.gather(score, 1, at), 0.0)
    dmine = torch.where(real, s.dweights, 0.0) * s.scale
    if s.renorm:
        total = mine.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
        dmine = (dmine - (dmine * mine).sum(-1, keepdim=True) / total) / total
    dscore = torch.zeros(rows, experts, device=at.device).scatter_add_(1, at, torch.where(real, dmine, 0.0))
    if s.scoring == "sigmoid":
        dlogits = dscore * score * (1.0 - score)
    else:
        dlogits = score * (dscore - (dscore * score).sum(-1, keepdim=True))
    return dlogits.to(s.logits.dtype)


PLAIN = {"add": _plain_add, "grads": _plain_grads, "route": _plain_route, "route_grad": _plain_route_grad}


# ------------------------------------------------------------------------------------------------ the state and a pass

@functools.lru_cache(maxsize=1)
def _framework() -> SimpleNamespace:
    from hibana_amd.kernels import adapters, ops
    return SimpleNamespace(adapters=adapters, ops=ops)


def _rank_of(case: dict, adapter: int) -> int:
    return max(1, case["rank"] >> adapter % 4) if case["ragged"] else case["rank"]


def _used(case: dict) -> list[int]:
    """The adapters that the requests of a case have between them: as many as there can be, spread over the pool."""
    n = case["adapters"]
    live = min(n, (case["runs"] or case["rows"]) - case["none"])
    return [i * n // live for i in range(live)] if live else []


def _lengths(case: dict) -> list[int]:
    """The rows of the requests: one each, or those of sequences of different lengths."""
    if not case["runs"]:
        return [1] * case["rows"]
    share = [1.0 + 0.75 * math.sin(2.0 + 5.0 * i) for i in range(case["runs"])]
    most = case["rows"] - case["runs"]
    lengths = [1 + int(most * v / sum(share)) for v in share]
    lengths[0] += case["rows"] - sum(lengths)
    return lengths


def _prepare_adapters(case: dict, s: SimpleNamespace, g: torch.Generator, seed: int) -> None:
    rows, k, n, rank, count, dtype = case["rows"], case["in"], case["out"], case["rank"], case["adapters"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    rng = np.random.default_rng(seed)
    lengths, used = _lengths(case), _used(case)
    live = len(lengths) - case["none"]
    owner = used + [used[i] for i in rng.integers(len(used), size=live - len(used))] if used else []
    owner = rng.permutation(np.array(owner + [-1] * case["none"], dtype=np.int64))
    s.index = torch.from_numpy(np.repeat(owner, lengths).astype(np.int32)).cuda()
    s.ranks = torch.tensor([_rank_of(case, i) for i in range(count)], dtype=torch.int32, device="cuda")
    s.scale = (32.0 / s.ranks).sqrt()
    s.x = (normal(rows, k) * torch.exp(0.5 * normal(k))).to(dtype)  # channels of different sizes, as behind a norm
    s.a = (normal(count, rank, k) / k ** 0.5).to(dtype)
    s.b = (normal(count, rank, n) * 0.1).to(dtype)  # a trained adapter's: its output a fraction of the projection's
    behind = torch.arange(rank, device="cuda")[None, :, None] >= s.ranks[:, None, None]
    s.a.masked_fill_(behind, 0.0)
    s.b.masked_fill_(behind, 0.0)
    if s.path == "add":
        s.y = normal(rows, n).to(dtype)
    else:
        s.dy = (normal(rows, n) * 0.02).to(dtype)
    if own:
        s.pool = _framework().adapters.Adapters(s.a, s.b, s.scale, s.ranks if case["ragged"] else None)


def _prepare_routing(case: dict, s: SimpleNamespace, g: torch.Generator) -> None:
    rows, experts = case["rows"], case["experts"]
    for key in ("topk", "scoring", "groups", "kept", "renorm", "scale"):
        setattr(s, key, case[key])
    lean = 0.7 * torch.randn(experts, device="cuda", generator=g)  # experts that are popular with every row
    logits = 1.5 * torch.randn(rows, experts, device="cuda", generator=g) + lean
    if case["masked"]:
        logits.masked_fill_(torch.rand(rows, experts, device="cuda", generator=g) < case["masked"], -math.inf)
        logits[0] = -math.inf
    s.logits = logits.to(TYPES[case["dtype"]])
    s.bias = None
    if case["bias"]:  # learnt so as to even the experts' loads out: against what makes them popular
        s.bias = (-lean + 0.1 * torch.randn(experts, device="cuda", generator=g)) * (0.1 if s.scoring == "sigmoid" else 0.5 / experts)
    s.slots = None
    if case["padded"]:
        s.slots = torch.ones(rows, dtype=torch.int32, device="cuda")
        s.slots[rows - case["padded"]:] = 0
    if s.path == "route_grad":
        s.ids, _ = _plain_route(s)
        s.dweights = 0.1 * torch.randn(rows, s.topk, device="cuda", generator=g)


def prepare(case: dict, seed: int) -> SimpleNamespace:
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(path=case["path"])
    if s.path in ("add", "grads"):
        _prepare_adapters(case, s, g, seed)
    else:
        _prepare_routing(case, s, g)
    return s


def run(s: SimpleNamespace):
    if not own:
        return PLAIN[s.path](s)
    f = _framework()
    if s.path == "add":
        return f.adapters.add(s.y, s.x, s.pool, s.index)
    if s.path == "grads":
        return f.adapters.grads(s.dy, s.x, s.pool, s.index)
    if s.path == "route":
        return f.ops.route_experts(s.logits, s.topk, s.scoring, bias=s.bias, groups=s.groups, kept=s.kept, renormalize=s.renorm, scale=s.scale, slots=s.slots)
    return f.ops.route_experts_grad(s.dweights, s.logits, s.ids, s.scoring, renormalize=s.renorm, scale=s.scale)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _exact_adapters(case: dict, s: SimpleNamespace):
    """An adapter at a time, on its own rows."""
    index = s.index.tolist()
    x = s.x.double()
    if s.path == "add":
        out = s.y.double()
    else:
        dy = s.dy.double()
        dx = torch.zeros_like(x)
        da, db = (torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (s.a, s.b))
    for i in sorted(set(index) - {-1}):
        rows = torch.tensor([r for r, j in enumerate(index) if j == i], device=x.device)
        rank = _rank_of(case, i)
        a, b, scale = s.a[i, :rank].double(), s.b[i, :rank].double(), float(s.scale[i])
        if s.path == "add":
            out[rows] += scale * torch.mm(torch.mm(x[rows], a.T), b)
        else:
            inner = scale * torch.mm(dy[rows], b.T)
            dx[rows] = torch.mm(inner, a)
            da[i, :rank] = torch.mm(inner.T, x[rows])
            db[i, :rank] = scale * torch.mm(torch.mm(x[rows], a.T).T, dy[rows])
    return out if s.path == "add" else (dx, da, db)


def _exact_route(s: SimpleNamespace):
    """Selections one after another, each the largest choice that is left."""
    logits = s.logits.double().cpu().numpy()
    rows, experts = logits.shape
    with np.errstate(over="ignore", invalid="ignore"):
        if s.scoring == "sigmoid":
            score = 1.0 / (1.0 + np.exp(-logits))
        else:
            e = np.exp(logits - np.maximum(logits.max(1, keepdims=True), -1e300))
            score = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    choice = score + (0.0 if s.bias is None else s.bias.double().cpu().numpy())
    choice[np.isneginf(logits)] = -np.inf
    every = np.arange(rows)
    if s.groups > 1:
        size = experts // s.groups
        parts = choice.reshape(rows, s.groups, size)
        first = parts.max(2)
        second = np.full_like(first, -np.inf) if size == 1 else np.partition(parts, size - 2, axis=2)[:, :, size - 2]
        total = first + np.where(np.isneginf(second), 0.0, second)
        barred = np.ones((rows, s.groups), dtype=bool)
        for _ in range(s.kept):
            at = np.argmax(np.where(barred, total, -np.inf), axis=1)  # (a group of -inf has nothing to choose from)
            barred[every, at] = False
        choice = np.where(np.repeat(barred, size, axis=1), -np.inf, choice)
    ids, weights = np.full((rows, s.topk), experts, dtype=np.int32), np.zeros((rows, s.topk))
    padded = np.zeros(rows, dtype=bool) if s.slots is None else s.slots.cpu().numpy() == 0
    for j in range(s.topk):
        at = np.argmax(choice, axis=1)
        real = ~np.isneginf(choice[every, at]) & ~padded
        ids[real, j], weights[real, j] = at[real], score[every, at][real]
        choice[every, at] = -np.inf
    if s.renorm:
        weights /= np.maximum(weights.sum(1, keepdims=True), 1e-300)
    return torch.from_numpy(ids).cuda(), torch.from_numpy(weights * s.scale).cuda()


def _exact_route_grad(s: SimpleNamespace) -> torch.Tensor:
    """By differentiation of the weights in 64 bits."""
    logits = s.logits.double().requires_grad_()
    real = s.ids < s.logits.shape[1]
    at = s.ids.long().clamp(max=s.logits.shape[1] - 1)
    masked = torch.isneginf(logits).all(1, keepdim=True)
    inside = torch.where(masked, torch.zeros_like(logits), logits)
    score = torch.sigmoid(inside) if s.scoring == "sigmoid" else torch.softmax(inside, -1)
    weights = torch.gather(score, 1, at) * real
    if s.renorm:
        weights = weights / (weights.sum(-1, keepdim=True) + (~real.any(-1, keepdim=True)).double())
    return torch.autograd.grad((weights * s.scale * s.dweights.double()).sum(), logits)[0]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s.path in ("add", "grads"):
        return _exact_adapters(case, s)
    return _exact_route(s) if s.path == "route" else _exact_route_grad(s)


# ------------------------------------------------------------------------------------------------ what a pass has to do

def work(case: dict) -> dict:
    """Rows in and out once, the matrices of each adapter in use once (their gradients whole, in 32 bits); the products of the
    rows that have an adapter. Routing: logits in, and ids and weights out or the logits' gradient; some operations a logit."""
    rows, size = case["rows"], TYPES[case["dtype"]].itemsize
    if case["path"] in ("add", "grads"):
        k, n = case["in"], case["out"]
        used = _used(case)
        ranks = sum(_rank_of(case, i) for i in used)
        live = 0 if not used else rows * (1.0 - case["none"] / (case["runs"] or rows))
        products = live * (ranks / max(1, len(used))) * 2.0 * (k + n)
        if case["path"] == "add":
            return {"bytes": size * (live * k + 2.0 * rows * n + ranks * (k + n)) + 4.0 * rows, "flops": products}
        return {"bytes": size * (rows * (2.0 * k + n) + ranks * (k + n)) + 4.0 * case["adapters"] * case["rank"] * (k + n) + 4.0 * rows, "flops": 3.0 * products}
    experts, topk = case["experts"], case["topk"]
    if case["path"] == "route":
        return {"bytes": rows * (size * experts + 8.0 * topk), "flops": 10.0 * rows * experts}
    dense = case["scoring"] == "softmax" and not case["renorm"]
    return {"bytes": rows * (size * experts * (2.0 if dense else 1.0) + (size + 8.0) * topk), "flops": rows * ((8.0 * experts if dense else 0.0) + 12.0 * topk)}
