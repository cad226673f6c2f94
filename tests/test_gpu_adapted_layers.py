"""Adapters and routing as the framework's linears and blocks run them: beside frozen linears of each format, through the dense MLP and the
gated experts' layer, and a training step in which adapters and router learn around frozen four-bit weights."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import adapters as oad, mxfp4_format as om, route_experts as oroute
from tests.util import random_experts

pytestmark = pytest.mark.gpu


def _mxfp4(n, k, seed, pairs=0):
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    g = torch.Generator().manual_seed(seed)
    return Mxfp4Linear(*(t.cuda() for t in om.quantize(torch.randn(n, k, generator=g) / k ** 0.5)), pairs=pairs).tile()


def _nvfp4(n, k, seed):
    from tests.test_gpu_nvfp4 import _linear, _matrix
    return _linear(*_matrix(n, k, seed), alpha=0.02, inv=0.25)


def _pool(k, n, seed, dtype=torch.bfloat16, count=3, rank=8):
    from hibana_amd.kernels import adapters
    g = torch.Generator().manual_seed(seed)
    return adapters.Adapters.from_pairs([(torch.randn(rank - i, k, generator=g) / k ** 0.5, torch.randn(n, rank - i, generator=g) * 0.3, 0.5 + i) for i in range(count)], dtype)


@pytest.mark.parametrize("make", [_nvfp4, _mxfp4])
@pytest.mark.parametrize("m", [1, 9, 300])
def test_adapted_linear(m, make):
    from hibana_amd.kernels import ops
    lin, pool = make(256, 384, 1), _pool(384, 256, 2)
    x = torch.randn(m, 384, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    index = (torch.arange(m) % 4 - 1).cuda()
    got, y = ops.adapted_linear(x, lin, pool, index), lin(x)
    case = tuple(t.cpu() for t in (y, x, pool.a, pool.b, pool.scale, pool.ranks, index))
    assert bool(((got.double().cpu() - oad.add(*case)).abs() <= oad.add_bound(*case)).all())
    assert torch.equal(got[index < 0], y[index < 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adapted_linear(x, lin, pool, index)
    for seed in range(3):
        x.copy_(torch.randn(m, 384, generator=torch.Generator().manual_seed(seed)).bfloat16())
        index.copy_(index.roll(1))
        graph.replay()
        assert torch.equal(out, ops.adapted_linear(x, lin, pool, index))
    with pytest.raises(ValueError):
        ops.adapted_linear(x, lin, _pool(384, 255, 2), index)


@pytest.mark.parametrize("m", [2, 40, 300])
@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
def test_dense_mlp(form, which, m):
    from hibana_amd.kernels import adapters, mxfp4, ops
    from hibana_amd.model.mlp import Mlp
    make = _nvfp4 if form == "nvfp4" else _mxfp4
    lins = make(512, 128, 4), make(128, 256, 5)
    pools = tuple(_pool(lin.in_features, lin.out_features, 6 + i) if on else None for i, (lin, on) in enumerate(zip(lins, which)))
    mlp = Mlp(*lins, adapters=pools)
    x = torch.randn(m, 128, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    index = (torch.arange(m) % 4 - 1).cuda()
    assert torch.equal(mlp(x), Mlp(*lins)(x))
    gate_up = lins[0](x)
    gate_up = gate_up if pools[0] is None else adapters.add(gate_up, x, pools[0], index)
    if form == "nvfp4":
        rows = h = ops.silu_and_mul(gate_up)
    else:
        h = ops.silu_mul_quant_mxfp4(gate_up)
        rows = mxfp4.dequantize(h, torch.bfloat16)
    y = lins[1](h)
    want = y if pools[1] is None else adapters.add(y, rows, pools[1], index)
    got = mlp(x, index=index)
    assert torch.equal(got, want)
    none = mlp(x, index=torch.full((m,), -1, device="cuda"))
    assert torch.equal(got[index < 0], none[index < 0]) and not torch.equal(got, none)


def test_dense_mlp_refusals():
    from hibana_amd.kernels import mxfp4
    from hibana_amd.model.mlp import Mlp
    lins = _mxfp4(512, 128, 4), _mxfp4(128, 256, 5)
    for bad in [(_pool(128, 512, 1),), (_pool(128, 256, 1), None), (None, _pool(128, 256, 1))]:
        with pytest.raises(ValueError):
            Mlp(*lins, adapters=bad)
    mlp = Mlp(*lins, adapters=(_pool(128, 512, 1), None))
    x = torch.randn(4, 128, device="cuda").bfloat16()
    with pytest.raises(ValueError):
        mlp(mxfp4.quantize(x), index=torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        mlp(x.float(), index=torch.zeros(4, dtype=torch.int32, device="cuda"))  # the pool's type


@pytest.mark.parametrize("m, mode", [(1, "decode"), (12, "verify"), (300, "prefill")])
@pytest.mark.parametrize("form", ["w3", "mxfp4"])
def test_gated_layer_with_a_routing_rule(form, m, mode):
    from hibana_amd.kernels import mxfp4_moe, ops, w3_moe
    from hibana_amd.model.flashnext_moe import MoeLayer
    e, hidden, inter, topk = 24, 256, 128, 4
    g = torch.Generator().manual_seed(m)
    router, gate = (torch.randn(e, hidden, generator=g) * 0.3).bfloat16().cuda(), (torch.randn(1, hidden, generator=g) * 0.05).cuda()
    rule = ops.Routing("sigmoid", (0.1 * torch.randn(e, generator=g)).cuda(), groups=6, kept=3, scale=2.5)
    if form == "w3":
        experts, shared = random_experts(e, hidden, inter, True, 1)[0], random_experts(1, hidden, inter, True, 2)[0]
        layer = MoeLayer(router, gate, experts, topk, shared=shared, routing=rule)
    else:
        held = [t.cuda() for i, shape in enumerate([(2 * inter, hidden), (hidden, inter)]) for t in om.quantize(torch.randn(e, *shape, generator=g) / 16)]
        experts = mxfp4_moe.Mxfp4Experts(*held)
        layer = MoeLayer(router, gate, experts, topk, shared_gate_up=_mxfp4(256, hidden, 3), shared_down=_mxfp4(hidden, 128, 4), routing=rule)
    x = torch.randn(m, hidden, generator=g).bfloat16().cuda()
    steps = 3 if mode == "verify" else 1
    slots = torch.ones(m // steps, dtype=torch.int32)
    if m > 1:
        slots[-1] = 0
    ctx = SimpleNamespace(mode=mode, slots=slots.cuda(), seq_slots=slots.cuda(), verify_steps=steps)
    ids, weights = layer.route(x, ctx)
    padded = slots.repeat_interleave(steps).eq(0).numpy() if mode != "prefill" else None
    want = oroute.choose(torch.mm(x, router.T).double().cpu().numpy(), topk, "sigmoid", rule.bias.double().cpu().numpy(), 6, 3, padded)
    assert np.array_equal(ids.cpu().numpy(), want)
    got = layer(x, ctx)
    if form == "w3":
        assert torch.equal(got, w3_moe.moe_layer(layer.w3, x, ids, weights, shared=layer.shared, gate_vec=layer.shared_gate_vec, experts_total=e))
    else:
        pairs = mxfp4_moe.mxfp4_moe(layer.mxfp4, x, ids, weights, pairs=True)
        assert torch.equal(got, ops.moe_combine_pairs(pairs, ids, weights, layer.shared_mlp(x), x, layer.shared_gate_vec, 0, e))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, ctx)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        assert torch.equal(out, layer(x, ctx))
    with pytest.raises(ValueError):
        MoeLayer(router, gate, layer.w3 if form == "w3" else experts, topk, routing=rule, keep=2, budget=8)


def test_a_training_step_around_frozen_weights():
    """A frozen MXFP4 projection with adapters beside it, and frozen routed experts behind a router that learns: loss = the sum of both outputs times fixed
    weights. The gradients of the adapters and of the router's weights against the formulas in 64 bits, on the values that the step has; then a step of descent,
    which the next forward pass reads from the same tensors."""
    from hibana_amd.kernels import adapters, mxfp4_moe, ops
    m, hidden, inter, e, topk, n = 90, 256, 96, 16, 3, 192
    g = torch.Generator().manual_seed(20)
    lin = _mxfp4(n, hidden, 21)
    held = [t.cuda() for shape in [(2 * inter, hidden), (hidden, inter)] for t in om.quantize(torch.randn(e, *shape, generator=g) / 16)]
    experts = mxfp4_moe.tile(mxfp4_moe.Mxfp4Experts(*held))
    a = torch.nn.Parameter((torch.randn(2, 8, hidden, generator=g) / 16).bfloat16().cuda())
    b = torch.nn.Parameter((torch.randn(2, 8, n, generator=g) * 0.1).bfloat16().cuda())
    router = torch.nn.Parameter((torch.randn(hidden, e, generator=g) / 16).cuda())
    pool = adapters.Adapters(a, b, 2.0)
    x = torch.randn(m, hidden, generator=g).bfloat16().cuda()
    index = (torch.arange(m) % 3 - 1).int().cuda()
    d_dense, d_routed = torch.randn(m, n, generator=g).bfloat16().cuda(), torch.randn(m, hidden, generator=g).cuda()

    def forward():
        dense = adapters.add(lin(x), x, pool, index)
        logits = x.float() @ router
        ids, weights = ops.route_experts(logits, topk, "sigmoid", scale=1.5)
        pairs = mxfp4_moe.mxfp4_moe(experts, x, ids, weights.detach(), pairs=True).view(m, topk, hidden)
        routed = (weights[..., None] * pairs).sum(1)
        return dense, logits, ids, pairs, (dense.float() * d_dense.float()).sum() + (routed * d_routed).sum()
    dense, logits, ids, pairs, loss = forward()
    loss.backward()
    case = (d_dense.cpu(), x.cpu(), a.detach().cpu(), b.detach().cpu(), torch.full((2,), 2.0), None, index.cpu())
    (_, da, db), (_, bound_a, bound_b) = oad.grads(*case), oad.grads_bound(*case)
    for leaf, want, bound in ((a, da, bound_a), (b, db, bound_b)):  # rounded once more, to the parameters' type
        assert bool(((leaf.grad.double().cpu() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
    dw = (pairs.double() * d_routed.double()[:, None]).sum(-1).cpu().numpy()
    dlogits = oroute.grad(dw, logits.detach().double().cpu().numpy(), ids.cpu().numpy(), "sigmoid", True, 1.5)
    want = x.double().cpu().T @ torch.from_numpy(dlogits)
    # dw: sums of 256 FP32 products; the routing's gradient 2^-16 of the largest |dw|; the product over 90 rows: 2^-12 of the magnitudes holds all of it
    size = x.double().cpu().abs().T @ (torch.from_numpy(np.abs(dlogits)) + 2.0 ** -4 * torch.from_numpy(np.abs(dw)).amax(1, keepdim=True))
    assert bool(((router.grad.double().cpu() - want).abs() <= 2.0 ** -12 * size).all())
    with torch.no_grad():
        for leaf in (a, b, router):
            leaf -= 1e-3 * leaf.grad
            leaf.grad = None
    again = forward()
    case = tuple(t.detach().cpu() for t in (lin(x), x, a, b)) + (torch.full((2,), 2.0), None, index.cpu())
    assert bool(((again[0].detach().double().cpu() - oad.add(*case)).abs() <= oad.add_bound(*case)).all()) and not torch.equal(again[0], dense)
