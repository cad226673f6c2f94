"""A pool whose tensors are given other memory, types or shapes behind its back, on the CPU: nothing is launched."""
import pytest
import torch

from hibana_amd.kernels import adapters, mxfp4

BF, F16 = torch.bfloat16, torch.float16


def _pool():
    pool = adapters.Adapters(torch.nn.Parameter(torch.ones(2, 4, 8, dtype=BF)), torch.nn.Parameter(torch.ones(2, 4, 6, dtype=BF)), torch.ones(2), torch.full((2,), 4, dtype=torch.int32))
    pool.struct()
    return pool


def test_another_type_at_the_same_addresses():
    pool = _pool()
    pool.room(300, 1)
    at = pool.a.data_ptr()
    pool.a.data, pool.b.data = pool.a.data.view(F16), pool.b.data.view(F16)
    struct = pool.struct()._obj
    assert pool.a.data_ptr() == at == struct.a and struct.type == mxfp4.TYPES[F16] != mxfp4.TYPES[BF]
    wide = torch.ones(2, 4, 8)
    pool.a.data, pool.b.data = wide, torch.ones(2, 4, 6)
    pool.struct(), pool.room(300, 1)
    pool.a.data = torch.ones(1)  # (frees nothing: `wide` holds the block)
    pool.a.data, pool.b.data = wide.view(BF)[..., :8].contiguous(), pool.b.data.view(BF)[..., :6].contiguous()
    assert pool.struct()._obj.type == mxfp4.TYPES[BF]
    fresh = adapters.Adapters(pool.a, pool.b, pool.scale, pool.ranks)
    assert pool.room(300, 1) == fresh.room(300, 1)


@pytest.mark.parametrize("name,change", [("a", lambda t: t.view(F16)), ("b", lambda t: t.view(F16)), ("ranks", lambda t: t.view(torch.float32)), ("scale", lambda t: t.view(torch.int32)),
                                         ("ranks", lambda t: t[:1]), ("scale", lambda t: t[:1]), ("scale", lambda t: t[:1].expand(2)), ("ranks", lambda t: t[:1].expand(2))])
def test_what_does_not_fit_is_refused(name, change):
    pool = _pool()
    held = getattr(pool, name)
    held.data = change(held.data)
    with pytest.raises(ValueError):
        pool.struct()


@pytest.mark.parametrize("m,k", [((1 << 24) + 1, 8), (1, (1 << 22) + 1)])
def test_sizes_past_the_library_s_are_refused_by_name(m, k):
    pool = adapters.Adapters(torch.zeros(1, 1, k), torch.zeros(1, 1, 6))
    for grads in (0, 1):
        with pytest.raises(ValueError, match="rows"):
            pool.room(m, grads)
