"""The microscaled four-bit operators as the framework's blocks run them: the dense MLP, the gated experts' layer with its shared expert,
the latent block on ReLU^2 experts. Each stage against the FP64 oracle on what the stage before it gave."""
from types import SimpleNamespace

import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # of a rounding, relative


def _weights(n, k, seed, stack=()):
    g = torch.Generator().manual_seed(seed)
    return om.quantize(torch.randn(*stack, n, k, generator=g) / k ** 0.5)


def _linear(held, pairs=0):
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    return Mxfp4Linear(*(t.cuda() for t in held), pairs=pairs).tile(release=True)


def _near(got, want, off, dtype=torch.bfloat16):
    """One rounding to `dtype` of a value that is off by `off` at most."""
    far = (got.double().cpu() - want).abs()
    bound = off * 1.001 + HALF_STEP[dtype] * 1.01 * (want.abs() + off) + 1e-30
    assert bool((far <= bound).all()), float((far / bound).max())


def _product(x64, held):
    """(x w^T, what an FP32 sum of its K products may be off by)."""
    w = om.dequantize(*held)
    return x64 @ w.T, w.shape[1] * 2.0 ** -24 * (x64.abs() @ w.abs().T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m, hidden, inter, pairs", [(1, 96, 32, 0), (4, 512, 256, 64), (16, 256, 416, 32), (77, 544, 160, 0), (200, 256, 512, 16)])
def test_dense_mlp(m, hidden, inter, pairs, dtype):
    from hibana_amd.kernels import mxfp4, ops
    from hibana_amd.model.mlp import Mlp
    gate_up, down = _weights(2 * inter, hidden, m), _weights(hidden, inter, m + 1)
    mlp = Mlp(_linear(gate_up, pairs), _linear(down))
    x = torch.randn(m, hidden, generator=torch.Generator().manual_seed(m + 2)).to(dtype).cuda()
    got = mlp(x)
    assert got.dtype == dtype and got.shape == (m, hidden)
    between = ops.mxfp4_linear(x, mlp.gate_up)
    _near(between, *_product(om.through(x.cpu()), gate_up), dtype)
    h = ops.silu_mul_quant_mxfp4(between, pairs)
    want_h = om.quantize(om.silu_mul(between.cpu(), pairs))
    assert torch.equal(h.codes.cpu(), want_h[0]) and torch.equal(h.scales.cpu(), want_h[1])
    _near(got, *_product(om.dequantize(*want_h), down), dtype)
    ready = mlp(mxfp4.quantize(x))
    assert ready.dtype == torch.bfloat16
    if dtype == torch.bfloat16:
        assert torch.equal(ready, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(x)
    for seed in range(3):
        x.copy_(torch.randn(m, hidden, generator=torch.Generator().manual_seed(seed)).to(dtype))
        graph.replay()
        want = mlp(x)
        assert torch.equal(out, want)
    empty = mlp(x[:0])
    assert empty.shape == (0, hidden) and empty.dtype == dtype


def test_dense_mlp_refuses_mixed_formats():
    from hibana_amd.model.mlp import Mlp
    other = SimpleNamespace(in_features=64, out_features=96, pairs=0, w3=None)
    with pytest.raises(ValueError):
        Mlp(_linear(_weights(128, 96, 1)), other)
    with pytest.raises(ValueError):
        Mlp(SimpleNamespace(in_features=96, out_features=128, pairs=0, w3=None), _linear(_weights(96, 64, 1)))
    with pytest.raises(ValueError):
        Mlp(_linear(_weights(128, 96, 1)), _linear(_weights(96, 128, 1)))


@pytest.mark.parametrize("m, mode", [(1, "decode"), (4, "decode"), (12, "verify"), (70, "prefill"), (1100, "prefill")])
def test_gated_layer(m, mode):
    """Router, routed experts, the shared expert on its linears, the gated combine; padded rows name no expert."""
    from hibana_amd.kernels import mxfp4_moe
    from hibana_amd.model.flashnext_moe import MoeLayer
    e, hidden, inter, topk = 24, 256, 96, 4
    fc1, fc2 = _weights(2 * inter, hidden, 1, (e,)), _weights(hidden, inter, 2, (e,))
    experts = mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*fc1, *fc2)))
    shared = _linear(_weights(256, hidden, 3)), _linear(_weights(hidden, 128, 4))
    g = torch.Generator().manual_seed(m)
    router, gate = (torch.randn(e, hidden, generator=g) * 0.3).bfloat16(), torch.randn(1, hidden, generator=g) * 0.05
    x = torch.randn(m, hidden, generator=g).bfloat16()
    layer = MoeLayer(router.cuda(), gate.cuda(), experts, topk, shared_gate_up=shared[0], shared_down=shared[1])
    assert layer.bytes == experts.bytes + 2 * router.numel() + shared[0].bytes + shared[1].bytes
    steps = 3 if mode == "verify" else 1
    slots = torch.ones(m // steps, dtype=torch.int32)
    if m > 1:
        slots[-1] = 0
    ctx = SimpleNamespace(mode=mode, slots=slots.cuda(), seq_slots=slots.cuda(), verify_steps=steps)
    xd = x.cuda()
    got = layer(xd, ctx)
    ids, w = (t.cpu() for t in layer.route(xd, ctx))
    pad = slots.repeat_interleave(steps) == 0
    if mode != "prefill":
        assert (ids[pad] == e).all()
    want, off = om.moe(x, ids, w, fc1, fc2)
    if m >= 1024:  # pairs in BF16
        y, pair_off = om.moe_pairs(x, ids, fc1, fc2)
        off = off + 2.0 ** -8 * ((y.abs() + pair_off) * w.double()[..., None]).sum(1)
    beside = MoeLayer(router.cuda(), gate.cuda(), experts, topk)
    assert beside.bytes == experts.bytes + 2 * router.numel()
    _near(beside(xd, ctx), want, off)
    # bf16(bf16(routed) + sigmoid(x . gate) shared): the dot off by H 2^-24 sum |x g|, which the sigmoid takes at a quarter at most
    lone = layer.shared_mlp(xd).double().cpu()
    products = x.double() * gate.double()
    open_ = torch.sigmoid(products.sum(-1, keepdim=True))
    moved = (hidden * 2.0 ** -24 * products.abs().sum(-1, keepdim=True) / 4 + 2.0 ** -20 * open_) * lone.abs()
    _near(got, want + open_ * lone, off + 2.0 ** -8 * (want.abs() + off) + moved + 2.0 ** -22 * (want.abs() + lone.abs()))
    assert torch.equal(got, layer(xd, ctx))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(xd, ctx)
    for seed in range(3):
        xd.copy_(torch.randn(m, hidden, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        assert torch.equal(out, layer(xd, ctx))


def test_gated_layer_of_a_range_of_the_experts():
    """Two ranks' parts add up to the whole sum, to their own roundings."""
    from hibana_amd.kernels import mxfp4_moe
    from hibana_amd.model.flashnext_moe import MoeLayer
    e, hidden, inter = 12, 128, 64
    fc1, fc2 = _weights(2 * inter, hidden, 5, (e,)), _weights(hidden, inter, 6, (e,))
    g = torch.Generator().manual_seed(7)
    router, gate, x = (torch.randn(e, hidden, generator=g) * 0.3).bfloat16().cuda(), torch.zeros(hidden).cuda(), torch.randn(9, hidden, generator=g).bfloat16()
    parts = []
    for lo in (0, 6):
        experts = mxfp4_moe.Mxfp4Experts(*(t[lo:lo + 6].contiguous().cuda() for t in (*fc1, *fc2)), base=lo)
        layer = MoeLayer(router, gate, experts, 3)
        ids, w = (t.cpu() for t in layer.route(x.cuda()))
        part = layer(x.cuda())
        half = [tuple(t[lo:lo + 6] for t in fc) for fc in (fc1, fc2)]
        _near(part, *om.moe(x, ids, w, *half, base=lo))
        parts.append(part.double().cpu())
    want, off = om.moe(x, ids, w, fc1, fc2)
    assert bool(((sum(parts) - want).abs() <= 2 * off + 2.0 ** -7 * sum(p.abs() for p in parts) + 1e-30).all())


def test_gated_layer_refusals():
    from hibana_amd.kernels import mxfp4_moe
    from hibana_amd.model.flashnext_moe import MoeLayer
    e, hidden, inter = 4, 128, 64
    make = lambda h_out=hidden, base=0: mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*_weights(2 * inter, hidden, 1, (e,)), *_weights(h_out, inter, 2, (e,)))), base=base)  # noqa: E731
    router, gate = torch.zeros(e, hidden, dtype=torch.bfloat16).cuda(), torch.zeros(hidden).cuda()
    up, down = _linear(_weights(128, hidden, 3)), _linear(_weights(hidden, 64, 4))
    for bad in [dict(experts=make(base=1)), dict(experts=make(h_out=160)), dict(shared_gate_up=up), dict(shared_gate_up=up, shared_down=SimpleNamespace(w3=None)),
                dict(shared=object()), dict(shared_gate_up=_linear(_weights(128, 96, 3)), shared_down=_linear(_weights(96, 64, 4)))]:
        with pytest.raises(ValueError):
            MoeLayer(**{**dict(router=router, shared_gate=gate, experts=make(), topk=2), **bad})


def test_weights_are_laid_out_ahead_of_a_capture():
    from hibana_amd.kernels import mxfp4_moe, ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    lin = Mxfp4Linear(*(t.cuda() for t in _weights(64, 96, 1)))
    experts = mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*_weights(64, 96, 1, (3,)), *_weights(96, 32, 2, (3,)))))
    x, ids, w = torch.zeros(2, 96, dtype=torch.bfloat16).cuda(), torch.zeros(2, 1, dtype=torch.int32).cuda(), torch.ones(2, 1).cuda()
    for call in (lambda: ops.mxfp4_linear(x, lin), lambda: mxfp4_moe.mxfp4_moe(experts, x, ids, w)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(graph):
                call()
    assert lin.tiled is None and experts.tiled1 is None
    assert not ops.mxfp4_linear(x, lin).any() and not mxfp4_moe.mxfp4_moe(experts, x, ids, w).any()  # and the calls go on


def test_latent_block_on_relu2_experts():
    """`NemotronMoe` with ReLU^2 experts of the format: its routed part is the operator's on the block's own routing."""
    from hibana_amd.kernels import mxfp4_moe
    from hibana_amd.model.nemotron_moe import NemotronMoe
    e, hidden, latent, inter, topk = 20, 192, 128, 96, 5
    fc1, fc2 = _weights(inter, latent, 8, (e,)), _weights(latent, inter, 9, (e,))
    g = torch.Generator().manual_seed(10)
    gate_fc1, back = (torch.randn(e + latent, hidden, generator=g) / hidden ** 0.5).bfloat16().cuda(), torch.randn(hidden, latent, generator=g).bfloat16().cuda()
    block = NemotronMoe(gate_fc1, torch.zeros(e).cuda(), back, mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*fc1, *fc2))), topk)
    for m in (1, 6, 50):
        x = torch.randn(m, hidden, generator=g).bfloat16().cuda()
        ids, w, lat = block.route(torch.mm(x, gate_fc1.T, out_dtype=torch.float32))
        routed = block.routed(lat, ids, w)
        _near(routed, *om.moe(lat.cpu(), ids.cpu(), w.cpu(), fc1, fc2))
        assert torch.equal(block(x), torch.mm(routed, back.T))
