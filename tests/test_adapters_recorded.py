"""What `adapters.add` records for its gradient, with the kernels replaced by their formulas on the CPU: nothing is launched."""
import pytest
import torch

from hibana_amd.kernels import adapters
from oracle import adapters as oracle


@pytest.fixture(autouse=True)
def formulas(monkeypatch):
    def add(y, x, pool, index, out):
        return oracle.add(y, x, pool.a, pool.b, pool.scale, pool.ranks, index).to(y.dtype)

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
