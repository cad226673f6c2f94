"""What the routing refuses, on the CPU: nothing is launched."""
import pytest
import torch

from hibana_amd import _lib
from hibana_amd.kernels import ops

CALL = dict(logits=256, type=2, stride=256, m=4, e=256, k=8, scoring=1, bias=256, groups=8, kept=4, renorm=1, scale=1.0, slots=256, steps=1, ids=256, weights=256, stream=None)
GRAD = dict(dweights=256, logits=256, type=0, stride=256, ids=256, m=4, e=256, k=8, scoring=1, renorm=1, scale=1.0, out=256, stream=None)


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(scoring=2), dict(m=0), dict(e=0), dict(e=1025, groups=1, kept=1, stride=2000), dict(k=0), dict(k=64), dict(k=33, kept=1), dict(groups=0),
                                    dict(groups=7), dict(groups=128, kept=4), dict(kept=0), dict(kept=9), dict(stride=255), dict(steps=0), dict(logits=258), dict(bias=258),
                                    dict(slots=258), dict(ids=258), dict(weights=258), dict(e=1023, groups=33, stride=1023)])
def test_calls(change):
    assert _lib.lib().hb_route_experts(*{**CALL, **change}.values()) == _lib.HB_EINVAL


@pytest.mark.parametrize("change", [dict(type=3), dict(scoring=-1), dict(m=0), dict(e=1025, stride=1025), dict(k=0), dict(k=64), dict(stride=255), dict(logits=257), dict(dweights=258), dict(ids=258),
                                    dict(out=264)])
def test_gradient_calls(change):
    assert _lib.lib().hb_route_experts_grad(*{**GRAD, **change}.values()) == _lib.HB_EINVAL


def test_missing():
    for key in ("logits", "ids", "weights"):
        assert _lib.lib().hb_route_experts(*{**CALL, key: None}.values()) == _lib.HB_ENULL
    for key in ("dweights", "logits", "ids", "out"):
        assert _lib.lib().hb_route_experts_grad(*{**GRAD, key: None}.values()) == _lib.HB_ENULL


def test_tensors():
    logits = torch.zeros(4, 32)
    for bad in [dict(logits=logits.double()), dict(logits=logits[0]), dict(k=0), dict(k=33), dict(k=17, groups=4, kept=2), dict(scoring="tanh"), dict(groups=5), dict(groups=4, kept=5), dict(kept=2),
                dict(bias=torch.zeros(31)), dict(bias=torch.zeros(1, 32)), dict(bias=torch.zeros(32, dtype=torch.int32)), dict(steps=0), dict(steps=3), dict(slots=torch.ones(3)), dict(slots=torch.ones(1), steps=2),
                dict(logits=torch.zeros(4, 1025)), dict(logits=torch.zeros(4, 0))]:
        it = dict(logits=logits, k=4, scoring="softmax", groups=1, kept=1) | bad
        with pytest.raises(ValueError):
            ops.route_experts(it.pop("logits"), it.pop("k"), it.pop("scoring"), **it)
    ids, dw = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    for bad in [(dw, logits.double(), ids), (dw, logits, ids.long()), (dw.half(), logits, ids), (dw[:3], logits, ids), (dw[:3], logits, ids[:3]), (dw[0], logits, ids[0])]:
        with pytest.raises(ValueError):
            ops.route_experts_grad(*bad)
    with pytest.raises(RuntimeError):
        ops.route_experts(logits, 4)
    with pytest.raises(RuntimeError):
        ops.route_experts_grad(dw, logits, ids)


def test_rows_past_what_a_launch_counts():
    assert _lib.lib().hb_route_experts(*{**CALL, "m": (1 << 25) + 1}.values()) == _lib.HB_EINVAL
    assert _lib.lib().hb_route_experts_grad(*{**GRAD, "m": (1 << 25) + 1}.values()) == _lib.HB_EINVAL
    with pytest.raises(ValueError, match="rows"):
        ops.route_experts(torch.empty((1 << 32) + 1, 1, dtype=torch.bfloat16, device="meta"), 1)
