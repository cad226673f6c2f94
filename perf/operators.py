"""The microscaled four-bit operators (MXFP4: E2M1 codes, two a byte, and one power-of-two scale, E8M0, for every 32
consecutive values of a row) as a served model calls them, from one decoded token to a prefill chunk.

Every case is a dict of plain values whose "path" names the operator:

  round    activations rounded to the format, and the values that the codes stand for: [rows, cols] of "dtype"
  silu     silu(gate) * up of a gate | up product [rows, 2 * cols] rounded to the format in the same pass; "pairs" > 0: gate
           and up alternate in blocks of that many columns
  linear   one projection: activations [rows, in] of "dtype" rounded to the format, times a weight [out, in] held in it
  moe      the routed experts of a layer: each row's "topk" experts, weighted and summed. "gated": silu(gate x) * (up x)
           between the two products, else relu(up x)^2; both products take their activations rounded to the format.
           "zipf": how uneven the experts' popularity is; "padded": that many last rows name no expert

The rounding of 32 values: the scale is 2^(floor(log2 of the largest magnitude) - 2), a value the nearest of 0, 1/2, 1, 3/2, 2,
3, 4 and 6 times it (ties to the even code, beyond 6 to 6).
"""
from __future__ import annotations

import functools
import math
from types import SimpleNamespace

import torch

own = False

GROUP = 32
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_FLOPS = 5.4e11  # of a drawn case: the largest listed one's
MOST_BYTES = 1.1e9


def listed() -> list[dict]:
    return [
        # one token's hidden state ahead of a projection: the smallest call
        {"name": "round_1", "path": "round", "rows": 1, "cols": 5120, "dtype": "bf16"},
        # a ragged prefill chunk whose residual stream is kept in 32 bits
        {"name": "round_f32_1543", "path": "round", "rows": 1543, "cols": 5120, "dtype": "f32"},
        # between a dense block's two products: four sequences decoding; a whole prefill chunk in fp16
        {"name": "silu_4", "path": "silu", "rows": 4, "cols": 25600, "pairs": 0, "dtype": "bf16"},
        {"name": "silu_f16_2048", "path": "silu", "rows": 2048, "cols": 25600, "pairs": 0, "dtype": "f16"},
        # one token through an attention-sized projection; an MLP's up projection for eight decoding sequences, for a ragged
        # verify batch, for a whole prefill chunk (the most arithmetic)
        {"name": "linear_1", "path": "linear", "rows": 1, "out": 5120, "in": 5120, "dtype": "bf16"},
        {"name": "linear_8", "path": "linear", "rows": 8, "out": 25600, "in": 5120, "dtype": "bf16"},
        {"name": "linear_f16_77", "path": "linear", "rows": 77, "out": 25600, "in": 5120, "dtype": "f16"},
        {"name": "linear_2048", "path": "linear", "rows": 2048, "out": 25600, "in": 5120, "dtype": "bf16"},
        # the routed layer: one token; four sequences verifying eight drafted tokens each, the last one padding; a ragged prefill
        # chunk (the most weights); ReLU^2 experts over a latent for four decoding sequences
        {"name": "moe_decode_1", "path": "moe", "rows": 1, "hidden": 2048, "inter": 512, "experts": 512, "topk": 10, "gated": True, "zipf": 0.0, "padded": 0},
        {"name": "moe_verify_32", "path": "moe", "rows": 32, "hidden": 2048, "inter": 512, "experts": 512, "topk": 10, "gated": True, "zipf": 1.1, "padded": 8},
        {"name": "moe_prefill_1543", "path": "moe", "rows": 1543, "hidden": 2048, "inter": 512, "experts": 512, "topk": 10, "gated": True, "zipf": 1.1, "padded": 0},
        {"name": "moe_relu2_4", "path": "moe", "rows": 4, "hidden": 1024, "inter": 2688, "experts": 512, "topk": 22, "gated": False, "zipf": 0.0, "padded": 0},
    ]


def _between(rng, low: float, high: float, step: int = 1) -> int:
    """A multiple of `step` between the two, spread evenly over the logarithm."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, int(round(value / step)) * step)


def draw(rng) -> dict:
    path = rng.choice(["round", "silu", "linear", "linear", "linear", "moe", "moe", "moe"])
    if path == "round":
        return {"path": path, "rows": _between(rng, 1, 2048), "cols": _between(rng, 32, 25600, 32), "dtype": rng.choice(list(TYPES))}
    if path == "silu":
        pairs = rng.choice([0, 0, 32, 64])
        return {"path": path, "rows": _between(rng, 1, 2048), "cols": _between(rng, 64, 25600, pairs or 32), "pairs": pairs, "dtype": rng.choice(list(TYPES))}
    if path == "linear":
        case = {"path": path, "rows": _between(rng, 1, 2048), "out": _between(rng, 64, 25600), "in": _between(rng, 256, 25600, 32), "dtype": rng.choice(list(TYPES))}
    else:
        rows = _between(rng, 1, 2048)
        gated = rng.random() < 0.7
        case = {"path": path, "rows": rows, "hidden": _between(rng, 512, 2560, 32), "inter": _between(rng, 256, 768 if gated else 2688, 32),
                "experts": _between(rng, 16, 512), "topk": rng.randint(2, 12 if gated else 16), "gated": gated, "zipf": rng.choice([0.0, 1.1]),
                "padded": rng.choice([0, 0, rows // 4])}
    while work(case)["flops"] > MOST_FLOPS or work(case)["bytes"] > MOST_BYTES:
        case["rows"] = case["rows"] * 3 // 4
    return case


# ------------------------------------------------------------------------------------------------ the plain form

def _power(byte: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) for E8M0 bytes (0 .. 254), as FP32."""
    bits = byte.to(torch.int32) << 23
    return torch.where(byte == 0, torch.full_like(bits, 1 << 22), bits).view(torch.float32)


def _rounded(x: torch.Tensor):
    """FP32 or FP64 [..., K] -> (values in units of the scale [..., K / 32, 32], E8M0 bytes [..., K / 32, 1])."""
    groups = x.unflatten(-1, (-1, GROUP))
    exponent = torch.frexp(groups.abs().amax(-1, keepdim=True)).exponent - 3  # |x| = m 2^e, 1/2 <= m < 1: floor(log2) is e - 1
    byte = (exponent + 127).clamp(0, 254)
    byte = torch.where(groups.abs().amax(-1, keepdim=True) == 0, torch.zeros_like(byte), byte)
    scaled = groups * _power(254 - byte).to(x.dtype)
    size = scaled.abs().clamp(max=6.0)
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0)).to(x.dtype)
    return torch.copysign(torch.round(size / step) * step, scaled), byte


def _through(x: torch.Tensor) -> torch.Tensor:
    """The values that x [..., K] rounded to the format stands for, FP32."""
    values, byte = _rounded(x)
    return (values.float() * _power(byte)).flatten(-2)


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Packed codes uint8 [..., K / 2] (element 2 i in the low nibble) and E8M0 scales [..., K / 32] -> FP32 [..., K]."""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (table[nibbles.int()].unflatten(-1, (-1, GROUP)) * _power(scales.int()).unsqueeze(-1)).flatten(-2)


def _gate_up(x: torch.Tensor, pairs: int):
    if not pairs:
        return x.chunk(2, -1)
    both = x.unflatten(-1, (-1, 2, pairs))
    return both[..., 0, :].flatten(-2), both[..., 1, :].flatten(-2)


def _plain_moe(s: SimpleNamespace) -> torch.Tensor:
    rows, topk = s.ids.shape
    experts = s.fc1[0].shape[0]
    ids = s.ids.reshape(-1).long()
    pair = torch.nonzero(ids < experts).squeeze(1)  # the pairs that name an expert, those of an expert behind one another
    used, which, count = torch.unique(ids[pair], return_inverse=True, return_counts=True)
    which, order = torch.sort(which, stable=True)
    pair = pair[order]
    place = torch.arange(len(pair), device=ids.device) - (count.cumsum(0) - count)[which]
    x = torch.zeros(len(used), int(count.max()), s.x.shape[1], device=ids.device)
    x[which, place] = _through(s.x.float())[pair // topk]
    y = torch.bmm(x, _values(*(t[used] for t in s.fc1)).transpose(1, 2).contiguous())
    if s.gated:
        up, gate = y.chunk(2, -1)
        h = gate / (1.0 + torch.exp(-gate)) * up
    else:
        h = torch.clamp(y, min=0.0).square()
    y = torch.bmm(_through(h), _values(*(t[used] for t in s.fc2)).transpose(1, 2).contiguous())
    of_pair = torch.zeros(rows * topk, y.shape[2], device=ids.device)
    of_pair[pair] = y[which, place]
    return (of_pair.unflatten(0, (rows, topk)) * s.weights.unsqueeze(-1)).sum(1).to(s.x.dtype)


def _plain(s: SimpleNamespace) -> torch.Tensor:
    if s.path == "round":
        return _through(s.x.float()).bfloat16()
    if s.path == "silu":
        gate, up = (t.double() for t in _gate_up(s.x, s.pairs))  # 64 bits: a product next to a border goes to its own side
        return _through(gate / (1.0 + torch.exp(-gate)) * up).bfloat16()
    if s.path == "linear":
        return (_through(s.x.float()) @ _values(*s.weight).T).to(s.x.dtype)
    return _plain_moe(s)


# ------------------------------------------------------------------------------------------------ the state and a pass

@functools.lru_cache(maxsize=1)
def _framework() -> SimpleNamespace:
    from hibana_amd.kernels import mxfp4, mxfp4_moe, ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    return SimpleNamespace(mxfp4=mxfp4, moe=mxfp4_moe, ops=ops, linear=Mxfp4Linear)


def _held(shape: tuple, g: torch.Generator):
    """A trained matrix's stand-in held in the format (normal values, an output of the order of one), a few matrices at a time."""
    def piece(n):
        w = torch.randn(n, *shape[1:], device="cuda", generator=g) / shape[-1] ** 0.5
        values, byte = _rounded(w)
        code = (torch.searchsorted(torch.tensor(LEVELS, device="cuda"), values.abs()) + 8 * (values < 0)).to(torch.uint8).flatten(-2)
        return code[..., 0::2] | code[..., 1::2] << 4, byte.squeeze(-1).to(torch.uint8)
    step = max(1, (1 << 27) // math.prod(shape[1:]))
    parts = [piece(min(step, shape[0] - at)) for at in range(0, shape[0], step)]
    return tuple(torch.cat(t) for t in zip(*parts))


def prepare(case: dict, seed: int) -> SimpleNamespace:
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(path=case["path"])
    rows, cols = case["rows"], {"round": "cols", "silu": "cols", "linear": "in", "moe": "hidden"}[case["path"]]
    cols = case[cols] * (2 if s.path == "silu" else 1)
    channel = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))  # channels of different sizes, as behind a norm
    s.x = (torch.randn(rows, cols, device="cuda", generator=g) * channel).to(TYPES[case.get("dtype", "bf16")])
    if s.path == "silu":
        s.pairs = case["pairs"]
    elif s.path == "linear":
        s.weight = _held((case["out"], cols), g)
        if own:  # the weights as a loader leaves them: laid out once
            s.weight = _framework().linear(*s.weight).tile(release=True)
    elif s.path == "moe":
        experts, inter, s.gated = case["experts"], case["inter"], case["gated"]
        popularity = -case["zipf"] * (torch.randperm(experts, device="cuda", generator=g) + 1.0).log()
        logits = popularity - torch.log(-torch.log(torch.rand(rows, experts, device="cuda", generator=g).clamp(1e-7, 1 - 1e-7)))
        top, ids = torch.topk(logits, case["topk"], dim=-1)
        s.weights, s.ids = torch.softmax(top, -1), ids.to(torch.int32)
        if case["padded"]:
            s.ids[-case["padded"]:], s.weights[-case["padded"]:] = experts, 0.0
        s.fc1 = _held((experts, 2 * inter if s.gated else inter, cols), g)  # gated: rows [up; gate]
        s.fc2 = _held((experts, cols, inter), g)
        if own:
            s.experts = _framework().moe.tile(_framework().moe.Mxfp4Experts(*s.fc1, *s.fc2), release=True)
            s.fc1 = s.fc2 = None
    return s


def run(s: SimpleNamespace) -> torch.Tensor:
    if not own:
        return _plain(s)
    f = _framework()
    if s.path == "round":
        return f.mxfp4.dequantize(f.mxfp4.quantize(s.x), torch.bfloat16)
    if s.path == "silu":
        return f.mxfp4.dequantize(f.ops.silu_mul_quant_mxfp4(s.x, s.pairs), torch.bfloat16)
    if s.path == "linear":
        return f.ops.mxfp4_linear(s.x, s.weight)
    return f.moe.mxfp4_moe(s.experts, s.x, s.ids, s.weights)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _nearest64(x: torch.Tensor) -> torch.Tensor:
    """FP64 [..., K] -> the values its rounding to the format stands for, FP64, by the borders between neighbouring levels."""
    groups = x.reshape(*x.shape[:-1], -1, GROUP)
    top = groups.abs().max(-1, keepdim=True).values
    _, e = torch.frexp(top)
    unit = torch.ldexp(torch.ones_like(top), torch.where(top == 0, -127, (e - 3).clamp(min=-127)))
    v = groups.abs() / unit
    out = 0.5 * (v > 0.25) + 0.5 * (v >= 0.75) + 0.5 * (v > 1.25) + 0.5 * (v >= 1.75) + (v > 2.5) * 1.0 + (v >= 3.5) * 1.0 + (v > 5.0) * 2.0
    return (torch.where(groups < 0, -out, out) * unit).reshape(x.shape)


def _values64(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    def value(c):
        sign, e, m = c >> 3, (c >> 1) & 3, c & 1
        size = torch.where(e == 0, 0.5 * m, torch.ldexp(1.0 + 0.5 * m.double(), e.int() - 1))
        return torch.where(sign == 1, -size, size)
    c = codes.long()
    both = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    both[..., 0::2], both[..., 1::2] = value(c % 16), value(c // 16)
    return both * torch.ldexp(torch.ones((), dtype=torch.float64, device=c.device), scales.int() - 127).repeat_interleave(GROUP, dim=-1)


def exact(case: dict, seed: int) -> torch.Tensor:
    s = prepare(case, seed)
    x = s.x.double()
    if s.path == "round":
        return _nearest64(x)
    if s.path == "silu":
        both = x.reshape(len(x), -1, 2, s.pairs or case["cols"])
        gate, up = both[:, :, 0].reshape(len(x), -1), both[:, :, 1].reshape(len(x), -1)
        return _nearest64(gate * torch.sigmoid(gate) * up)
    x = _nearest64(x)
    if s.path == "linear":
        pieces = [x @ _values64(s.weight[0][at:at + 4096], s.weight[1][at:at + 4096]).T for at in range(0, case["out"], 4096)]
        return torch.cat(pieces, 1)
    out = torch.zeros_like(x)
    inter = case["inter"]
    for e in torch.unique(s.ids).tolist():
        if e >= case["experts"]:
            continue
        row, slot = torch.nonzero(s.ids == e, as_tuple=True)
        y = x[row] @ _values64(s.fc1[0][e], s.fc1[1][e]).T
        h = y[:, inter:] * torch.sigmoid(y[:, inter:]) * y[:, :inter] if s.gated else y * y * (y > 0)
        out[row] += s.weights[row, slot].double()[:, None] * (_nearest64(h) @ _values64(s.fc2[0][e], s.fc2[1][e]).T)
    return out


# ------------------------------------------------------------------------------------------------ what a pass has to do

def _distinct(rows: int, experts: int, topk: int, zipf: float) -> float:
    """The experts that `rows` draws of `topk` name, on average: one is in a row's top k with a probability that grows with
    its popularity, the probabilities adding up to topk."""
    p = [(e + 1.0) ** -zipf for e in range(experts)]
    low, high = 0.0, 1e9
    for _ in range(100):
        mid = math.sqrt(low * high) if low else high / 2
        low, high = (mid, high) if sum(1.0 - math.exp(-mid * v) for v in p) < topk else (low, mid)
    return sum(1.0 - math.exp(-high * v * rows) for v in p)


def _matrix_bytes(n: float, k: float) -> float:
    return n * k / 2 + n * k / GROUP


def work(case: dict) -> dict:
    """Activations in and results out once, each weight that is named once; the products of the rows that name an expert, and
    eight operations for a rounded value."""
    rows = case["rows"]
    size = TYPES[case.get("dtype", "bf16")].itemsize
    if case["path"] == "round":
        return {"bytes": rows * case["cols"] * (size + 2.0), "flops": 8.0 * rows * case["cols"]}
    if case["path"] == "silu":
        return {"bytes": rows * case["cols"] * (2.0 * size + 2.0), "flops": 12.0 * rows * case["cols"]}
    if case["path"] == "linear":
        n, k = case["out"], case["in"]
        return {"bytes": _matrix_bytes(n, k) + size * rows * (n + k), "flops": 2.0 * rows * n * k}
    h, i, n1 = case["hidden"], case["inter"], case["inter"] * (2 if case["gated"] else 1)
    real = rows - case["padded"]
    distinct = _distinct(real, case["experts"], case["topk"], case["zipf"])
    return {"bytes": distinct * (_matrix_bytes(n1, h) + _matrix_bytes(h, i)) + rows * (4.0 * h + 8.0 * case["topk"]),
            "flops": 2.0 * real * case["topk"] * h * (n1 + i)}
