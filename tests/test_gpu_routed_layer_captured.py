"""The gated experts' layer with a routing rule serves whatever its router is: a parameter that takes a gradient too, called eagerly and captured."""
import pytest
import torch

from oracle import mxfp4_format as om
from tests.test_gpu_adapted_layers import _mxfp4
from tests.util import random_experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["w3", "mxfp4", "mxfp4 shared"])
def test_a_router_that_is_a_parameter(form):
    from hibana_amd.kernels import mxfp4_moe, ops
    from hibana_amd.model.flashnext_moe import MoeLayer
    e, hidden, inter, m = 16, 256, 128, 9
    g = torch.Generator().manual_seed(3)
    held, gate = (torch.randn(e, hidden, generator=g) * 0.3).bfloat16().cuda(), torch.zeros(1, hidden, device="cuda")
    rule = ops.Routing("sigmoid", scale=2.0)
    if form == "w3":
        experts, more = random_experts(e, hidden, inter, True, 1)[0], dict(shared=random_experts(1, hidden, inter, True, 2)[0])
    else:
        experts = mxfp4_moe.Mxfp4Experts(*[t.cuda() for shape in [(2 * inter, hidden), (hidden, inter)] for t in om.quantize(torch.randn(e, *shape, generator=g) / 16)])
        more = dict(shared_gate_up=_mxfp4(256, hidden, 3), shared_down=_mxfp4(hidden, 128, 4)) if "shared" in form else {}
    layer = MoeLayer(torch.nn.Parameter(held), gate, experts, 3, routing=rule, **more)
    x = torch.randn(m, hidden, generator=g).bfloat16().cuda()
    with torch.no_grad():
        want = layer(x)
    got = layer(x)
    assert torch.equal(got, want) and not got.requires_grad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        with torch.no_grad():
            assert torch.equal(out, layer(x))
    ids, weights = layer.route(x)  # called by itself, the routing records its gradient
    weights.sum().backward()
    assert layer.router.grad is not None
