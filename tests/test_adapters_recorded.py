"""What `adapters.add` records for its gradient, with the kernels replaced by their formulas on the CPU: nothing is launched."""
import pytest
import torch

from hibana_amd.kernels import adapters
from oracle import adapters as oracle


@pytest.fixture(autouse=True)
def formulas(monkeypatch):
    def add(y, x, pool, index, out):
        to = oracle.add(y, x, pool.a, pool.b, pool.scale, pool.ranks, index).to(y.dtype)
        return to if out is None else (out.data.copy_(to), out)[1]  # (as a kernel writes it: past autograd)

    def grads(dy, x, pool, index):
        dx, da, db = oracle.grads(dy, x, pool.a, pool.b, pool.scale, pool.ranks, index)
        return dx.to(x.dtype), da.float(), db.float()
    monkeypatch.setattr(adapters, "_add", add)
    monkeypatch.setattr(adapters, "grads", grads)


def _case(ranks=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    pool = adapters.Adapters(torch.nn.Parameter(torch.randn(3, 4, 8, generator=g)), torch.nn.Parameter(torch.randn(3, 4, 6, generator=g)), torch.tensor([0.5, 1.0, 2.0]),
                             torch.tensor([4, 2, 3], dtype=torch.int32) if ranks else None)
    y, x, dy = (torch.randn(5, n, generator=g).requires_grad_(n != 7) for n in (6, 8, 6))
    return pool, y, x, dy.detach(), torch.tensor([0, 1, -1, 2, 1])


def _gradients(pool, y, x):
    got = [t.grad for t in (y, x, pool.a, pool.b)]
    for t in (y, x, pool.a, pool.b):
        t.grad = None
    return got


@pytest.mark.parametrize("ranks", [True, False])
def test_a_scale_or_a_rank_put_in_the_old_one_s_place_is_the_next_call_s(ranks):
    """The gradient is that of the function that the forward pass computed."""
    pool, y, x, dy, index = _case(ranks)
    adapters.add(y, x, pool, index).backward(dy)
    want = _gradients(pool, y, x)
    out = adapters.add(y, x, pool, index)
    pool.scale = pool.scale * 3
    pool.ranks = torch.ones(3, dtype=torch.int32)
    out.backward(dy)
    for got, w in zip(_gradients(pool, y, x), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("name", ["scale", "ranks", "a", "b"])
def test_a_change_in_place_is_noticed(name):
    pool, y, x, dy, index = _case()
    out = adapters.add(y, x, pool, index)
    with torch.no_grad():
        getattr(pool, name).mul_(2 if name != "ranks" else 0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dy)


def test_an_adapter_set_between_the_passes_is_noticed():
    pool, y, x, dy, index = _case()
    out = adapters.add(y, x, pool, index)
    pool.set(1, torch.ones(1, 8), torch.ones(6, 1), 3.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dy)


def test_several_passes_at_scales_of_their_own():
    pool, y, x, dy, index = _case()
    first = adapters.add(y, x, pool, index)
    pool.scale = pool.scale * 3
    second = adapters.add(y, x, pool, index)
    pool.scale = pool.scale / 3
    (first.mul(dy).sum() + second.mul(dy).sum()).backward()
    got = _gradients(pool, y, x)
    adapters.add(y, x, pool, index).backward(dy)
    once = _gradients(pool, y, x)
    torch.testing.assert_close(got[2], 4 * once[2])
    torch.testing.assert_close(got[3], 4 * once[3])


def test_a_scale_that_begins_to_take_a_gradient_is_refused():
    pool, y, x, _, index = _case()
    pool.scale.requires_grad_()
    with pytest.raises(ValueError, match="scale"):
        adapters.add(y, x, pool, index)


def test_a_projection_without_a_gradient_beside_rows_with_one_is_refused():
    """y of a frozen linear's kernels records nothing: x's gradient would lack the projection's own part, dy W, and a layer below would learn from the rest."""
    pool, y, x, dy, index = _case()
    with pytest.raises(ValueError, match="dy W"):
        adapters.add(y.detach(), x, pool, index)
    adapters.add(y.detach(), x.detach(), pool, index).backward(dy)  # the lowest adapted layer
    da = pool.a.grad.clone()
    with torch.no_grad():
        assert not adapters.add(y.detach(), x, pool, index).requires_grad
    adapters.add(y.detach().requires_grad_(), x, pool, index).backward(dy)  # the caller's own dy W beside it
    assert x.grad is not None and torch.equal(pool.a.grad, 2 * da)


def test_two_adapted_layers_learn_through_a_projection_that_records_its_gradient():
    """The layers' frozen projections as a function of the program's own (dx = dy W), against differences of the loss in the lower layer's adapters."""
    class Frozen(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(w)
            return x @ w.T

        @staticmethod
        def backward(ctx, dy):
            return dy @ ctx.saved_tensors[0], None
    g = torch.Generator().manual_seed(2)
    normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    low, high = (adapters.Adapters(torch.nn.Parameter(normal(2, 3, 8)), torch.nn.Parameter(normal(2, 3, 8))) for _ in range(2))
    w0, w1, x, dy, index = normal(8, 8), normal(8, 8), normal(5, 8), normal(5, 8), torch.tensor([0, 1, -1, 1, 0])

    def loss(low, high, x, w0, w1, dy):
        h = adapters.add(x @ w0.T, x, low, index)
        return (adapters.add(Frozen.apply(h, w1), h, high, index) * dy).sum()
    args = (x, w0, w1, dy)
    loss(low, high, *args).backward()
    grad, step = low.a.grad.clone(), torch.sign(normal(2, 3, 8))
    with torch.no_grad():
        ends = [loss(adapters.Adapters(low.a + s * step, low.b), high, *args).double() for s in (0.5, -0.5)]
        # linear in low.a, so the difference is the gradient but for FP32's roundings: at most 8 + 1 + 8 + 1 of them behind one another, 40 more in the sum
        size = loss(adapters.Adapters(low.a.abs() + 0.5, low.b.abs()), adapters.Adapters(high.a.abs(), high.b.abs()), *(t.abs() for t in args)).item()
    assert abs((ends[0] - ends[1]).item() - (grad.double() * step).sum().item()) <= 4 * 58 * 2.0 ** -24 * size


def test_a_result_put_into_a_tensor_is_a_change_of_it():
    """Who keeps the old values for a gradient is told, as by any operation in place; on tensors of inference mode there is nobody to tell."""
    pool, y, x, _, index = _case()
    y, weight = y.detach(), torch.ones(6, requires_grad=True)
    kept = (weight * y).sum()
    at = y._version
    with torch.no_grad():
        assert adapters.add(y, x, pool, index, out=y) is y
    assert y._version > at
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    with torch.inference_mode():
        z = y.clone()
        assert adapters.add(z, x, pool, index, out=z) is z and not torch.equal(z, y)
