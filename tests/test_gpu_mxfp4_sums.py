"""The weighted sums of routed experts in the microscaled four-bit format at prefill sizes: FP32 pairs, one rounding, whatever the number of rows."""
from types import SimpleNamespace

import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu


def _stack(e, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return om.quantize(torch.randn(e, n, k, generator=g) / k ** 0.5)


def _inputs(m, e, k, hidden, seed):
    g = torch.Generator().manual_seed(seed)
    w, ids = torch.topk(torch.randn(m, e, generator=g), k, dim=-1)
    return torch.randn(m, hidden, generator=g).bfloat16(), ids.to(torch.int32), torch.softmax(w, -1)


def _check(got, want, off):
    """`off` and the one rounding to BF16 (half a step, 2^-8 of the value)."""
    far = (got.double().cpu() - want).abs()
    bound = off * 1.001 + 2.0 ** -8 * 1.01 * (want.abs() + off) + 1e-30
    assert bool((far <= bound).all()), float((far / bound).max())


# rows, experts, top k, hidden, inter, gated: below and from the size at which the framework's three-bit calls keep BF16 pairs; 20 and 48 pairs an expert
# (slots of 32 and of 64 rows), 400 (the ring)
SIZES = [(1023, 64, 3, 64, 96, True), (1024, 200, 4, 64, 96, True), (1100, 64, 3, 96, 64, False), (1030, 11, 4, 512, 512, True)]


@pytest.mark.parametrize("m, e, k, hidden, inter, gated", SIZES)
def test_sums_are_rounded_once(m, e, k, hidden, inter, gated):
    from hibana_amd.kernels import mxfp4_moe
    fc1, fc2 = _stack(e, 2 * inter if gated else inter, hidden, m), _stack(e, hidden, inter, m + 1)
    ex = mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*fc1, *fc2)))
    x, ids, w = _inputs(m, e, k, hidden, m + 2)
    want, off = om.moe(x, ids, w, fc1, fc2)
    args = ex, x.cuda(), ids.cuda(), w.cuda()
    got = mxfp4_moe.mxfp4_moe(*args)
    _check(got, want, off)
    for _ in range(3):
        assert torch.equal(got, mxfp4_moe.mxfp4_moe(*args))


def test_pairs_beside_a_shared_expert_are_not_rounded():
    """The layer's combine takes FP32 pairs: with a shared expert whose gate is shut the result is the routed sum's."""
    from hibana_amd.kernels import mxfp4_moe
    from hibana_amd.model.flashnext_moe import MoeLayer
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    m, e, topk, hidden, inter = 1100, 64, 3, 128, 64
    fc1, fc2 = _stack(e, 2 * inter, hidden, 1), _stack(e, hidden, inter, 2)
    experts = mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*fc1, *fc2)))
    x, _, _ = _inputs(m, e, topk, hidden, 3)
    x[:, 0] = 1.0
    gate = torch.zeros(hidden)
    gate[0] = -200.0  # sigmoid(-200) is nothing in FP32
    router = (torch.randn(e, hidden, generator=torch.Generator().manual_seed(4)) * 0.3).bfloat16()
    shared = [Mxfp4Linear(*(t[0].cuda() for t in _stack(1, n, k, n))) for n, k in ((128, hidden), (hidden, 64))]
    layer = MoeLayer(router.cuda(), gate.cuda(), experts, topk, shared_gate_up=shared[0], shared_down=shared[1])
    ctx = SimpleNamespace(mode="prefill", slots=torch.ones(m, dtype=torch.int32, device="cuda"), seq_slots=torch.ones(m, dtype=torch.int32, device="cuda"), verify_steps=1)
    got = layer(x.cuda(), ctx)
    ids, w = (t.cpu() for t in layer.route(x.cuda(), ctx))
    want, off = om.moe(x, ids, w, fc1, fc2)
    # bf16(bf16(routed) + 0): the second rounding changes nothing
    _check(got, want, off)
