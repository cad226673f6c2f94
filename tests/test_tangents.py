"""Forward-mode tangents: the adapters' and the routing's calls hold none, and refuse inputs that carry one, on the CPU: nothing is launched."""
import pytest
import torch
from torch.autograd import forward_ad

from hibana_amd.kernels import adapters, ops


def _args():
    pool = adapters.Adapters(torch.ones(2, 4, 8), torch.ones(2, 4, 6), torch.ones(2))
    return pool, torch.ones(3, 6), torch.ones(3, 8), torch.zeros(3, dtype=torch.int32)


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["y", "x", "a", "b", "scale"])
def test_adapters(which, grad):
    pool, y, x, index = _args()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        if which in ("a", "b", "scale"):
            setattr(pool, which, _dual(getattr(pool, which)))
        y, x = _dual(y) if which == "y" else y, _dual(x) if which == "x" else x
        with pytest.raises(NotImplementedError, match="tangent"):
            adapters.add(y, x, pool, index)
        with pytest.raises(NotImplementedError, match="tangent"):
            adapters.grads(y, x, pool, index)


@pytest.mark.parametrize("grad", [True, False])
def test_routing(grad):
    logits, ids, dw = torch.ones(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, 2)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="tangent"):
            ops.route_experts(_dual(logits), 2)
        with pytest.raises(NotImplementedError, match="tangent"):
            ops.route_experts_grad(dw, _dual(logits), ids)
        with pytest.raises(NotImplementedError, match="tangent"):
            ops.route_experts_grad(_dual(dw), logits, ids)


def test_a_level_without_tangents():
    pool, y, x, index = _args()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="GPU only"):
            adapters.add(y, x, pool, index)
        with pytest.raises(RuntimeError, match="GPU only"):
            ops.route_experts(torch.ones(3, 8), 2)
