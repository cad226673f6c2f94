"""What the adapters refuse, on the CPU: nothing is launched."""
import ctypes as C
import copy
import pickle

import pytest
import torch

from hibana_amd import _lib
from hibana_amd.kernels import adapters

GOOD = dict(a=256, b=256, scale=256, ranks=256, adapters=4, rank=8, k=64, n=32, type=0)


def _struct(**change):
    return C.byref(_lib.HbAdapters(*{**GOOD, **change}.values()))


CALL = dict(x=256, x_stride=64, y=256, y_stride=32, index=256, index_bytes=4, m=10, out=512, out_stride=32, ws=1024, ws_bytes=1 << 30, stream=None)
GRADS = dict(x=256, x_stride=64, dy=256, dy_stride=32, index=256, index_bytes=4, m=10, dx=512, da=512, db=512, ws=1024, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(adapters=0), dict(adapters=4097), dict(rank=0), dict(rank=257), dict(k=0), dict(n=-1), dict(k=(1 << 22) + 1),
                                    dict(a=257), dict(b=257), dict(scale=258), dict(ranks=258)])
def test_pools(change):
    lib = _lib.lib()
    assert lib.hb_adapters_add(_struct(**change), *CALL.values()) == _lib.HB_EINVAL
    assert lib.hb_adapters_grads(_struct(**change), *GRADS.values()) == _lib.HB_EINVAL
    if not {"a", "b", "scale", "ranks"} & set(change):
        assert lib.hb_adapters_workspace_bytes(_struct(**change), 10, 0) == lib.hb_adapters_workspace_bytes(_struct(**change), 10, 1) == 0


@pytest.mark.parametrize("change", [dict(m=0), dict(m=-1), dict(m=(1 << 24) + 1), dict(x_stride=63), dict(x_stride=1 << 31), dict(index_bytes=2), dict(index=258), dict(x=257), dict(ws=1032)])
def test_rows(change):
    lib = _lib.lib()
    assert lib.hb_adapters_add(_struct(), *{**CALL, **change}.values()) == _lib.HB_EINVAL
    assert lib.hb_adapters_grads(_struct(), *{**GRADS, **change}.values()) == _lib.HB_EINVAL


@pytest.mark.parametrize("change", [dict(y_stride=31), dict(out_stride=31), dict(out=257), dict(y=257), dict(y=512, y_stride=40)])
def test_rows_of_add(change):
    assert _lib.lib().hb_adapters_add(_struct(), *{**CALL, **change}.values()) == _lib.HB_EINVAL


@pytest.mark.parametrize("change", [dict(dy_stride=31), dict(dy=257), dict(dx=257), dict(da=258), dict(db=258)])
def test_rows_of_grads(change):
    assert _lib.lib().hb_adapters_grads(_struct(), *{**GRADS, **change}.values()) == _lib.HB_EINVAL


def test_missing_and_small():
    lib = _lib.lib()
    for key in ("x", "y", "index", "out", "ws"):
        assert lib.hb_adapters_add(_struct(), *{**CALL, key: None}.values()) == _lib.HB_ENULL
    for key in ("x", "dy", "index", "dx", "da", "db", "ws"):
        assert lib.hb_adapters_grads(_struct(), *{**GRADS, key: None}.values()) == _lib.HB_ENULL
    for key in ("a", "b"):
        assert lib.hb_adapters_add(_struct(**{key: None}), *CALL.values()) == _lib.HB_ENULL
    assert lib.hb_adapters_add(None, *CALL.values()) == _lib.HB_ENULL and lib.hb_adapters_workspace_bytes(None, 10, 0) == 0
    for call, grads, fn in ((CALL, 0, lib.hb_adapters_add), (GRADS, 1, lib.hb_adapters_grads)):
        need = lib.hb_adapters_workspace_bytes(_struct(), 1000, grads)
        assert need >= (1 + grads) * 1000 * 8 * 4
        assert fn(_struct(), *{**call, "m": 1000, "ws_bytes": need - 1}.values()) == _lib.HB_EWORKSPACE


def test_workspaces_hold_every_count_of_partial_sums():
    """An adapter of more than one unit of rows has a slot for each; whatever the split of the rows, they fit: the sizes grow with the rows and the pool."""
    lib = _lib.lib()
    sizes = [lib.hb_adapters_workspace_bytes(_struct(adapters=n, rank=r, k=512, n=512), m, 1) for m in (1, 300, 5000, 100000) for n in (1, 64, 4096) for r in (1, 16, 256)]
    assert all(sizes) and lib.hb_adapters_workspace_bytes(_struct(adapters=4096, rank=256, k=512, n=512), 1, 1) < 1 << 20  # (nothing the size of the pool)


def test_tensors():
    bf = torch.bfloat16
    a, b = torch.zeros(2, 4, 8, dtype=bf), torch.zeros(2, 4, 6, dtype=bf)
    pool = adapters.Adapters(a, b, 0.5)
    assert pool.scale.tolist() == [0.5, 0.5] and (pool.adapters, pool.rank, pool.in_features, pool.out_features, pool.bytes) == (2, 4, 8, 6, 2 * 4 * 14 * 2)
    for bad in [(a[0], b[0]), (a, b.float()), (a, b[:1]), (a, b[:, :3]), (a.double(), b.double()), (a, b, torch.ones(3)), (a, b, torch.ones(2).double()),
                (a, b, None, torch.ones(2)), (a, b, None, torch.ones(1, dtype=torch.int32)), (torch.zeros(2, 4, 16, dtype=bf)[..., ::2], b), (torch.zeros(2, 257, 8, dtype=bf), torch.zeros(2, 257, 6, dtype=bf)),
                (torch.zeros(4097, 1, 1, dtype=bf), torch.zeros(4097, 1, 1, dtype=bf)), (a[:0], b[:0])]:
        with pytest.raises(ValueError):
            adapters.Adapters(*bad)
    y, x, index = torch.zeros(3, 6, dtype=bf), torch.zeros(3, 8, dtype=bf), torch.zeros(3, dtype=torch.int32)
    for bad in [(y.float(), x, index), (y, x.half(), index), (y[:2], x, index), (y, x[:, :7], index), (y[None], x, index), (y, x, index[:2]), (y, x, index.float()), (y, x, index[None]),
                (y, x, index.bool()), (y, x, index.to(torch.int16))]:
        with pytest.raises(ValueError):
            adapters.add(bad[0], bad[1], pool, bad[2])
        with pytest.raises(ValueError):
            adapters.grads(bad[0], bad[1], pool, bad[2])
    with pytest.raises(RuntimeError):
        adapters.add(y, x, pool, index)  # CPU tensors: there is no fallback
    with pytest.raises(RuntimeError):
        adapters.grads(y, x, pool, index)


def test_pairs():
    pairs = [(torch.ones(2, 8), torch.ones(6, 2), 1.0), (torch.ones(3, 8), torch.ones(6, 3), 2.0)]
    pool = adapters.Adapters.from_pairs(pairs, torch.float32, "cpu")
    assert pool.ranks.tolist() == [2, 3] and pool.scale.tolist() == [1.0, 2.0] and pool.a[0, 2].eq(0).all() and pool.a[1].eq(1).all() and pool.b.shape == (2, 3, 6)
    for bad in [[], [(torch.ones(2, 8), torch.ones(6, 3), 1.0)], [pairs[0], (torch.ones(2, 7), torch.ones(6, 2), 1.0)], [pairs[0], (torch.ones(2, 8), torch.ones(5, 2), 1.0)]]:
        with pytest.raises(ValueError):
            adapters.Adapters.from_pairs(bad, torch.float32, "cpu")
    for bad in [(2, *pairs[0]), (-1, *pairs[0]), (0, torch.ones(4, 8), torch.ones(6, 4), 1.0), (0, torch.ones(2, 8), torch.ones(6, 3), 1.0), (0, torch.ones(2, 9), torch.ones(6, 2), 1.0)]:
        with pytest.raises(ValueError):
            pool.set(*bad)
    plain = adapters.Adapters(torch.zeros(2, 3, 8), torch.zeros(2, 3, 6))
    plain.set(1, *pairs[1][:2])
    for bad in [(0, *pairs[0][:2]), (1, *pairs[1])]:  # a lower rank, a scale: the pool holds neither
        with pytest.raises(ValueError):
            plain.set(*bad)


def test_a_pool_can_be_copied_and_pickled():
    pool = adapters.Adapters.from_pairs([(torch.ones(2, 8), torch.ones(6, 2), 1.0)], torch.float32, "cpu")
    pool.struct()
    for twin in (copy.copy(pool), copy.deepcopy(pool), pickle.loads(pickle.dumps(pool))):
        assert torch.equal(twin.a, pool.a) and twin.struct()._obj.a == twin.a.data_ptr()


def test_a_tensor_put_in_another_s_place_is_looked_at():
    pool = adapters.Adapters(torch.zeros(2, 3, 8), torch.zeros(2, 3, 6), 1.0)
    pool.struct()
    for name, bad in [("a", torch.zeros(2, 4, 8)), ("b", torch.zeros(2, 3, 12)[..., ::2]), ("scale", torch.zeros(3)), ("ranks", torch.zeros(2))]:
        kept = getattr(pool, name)
        setattr(pool, name, bad)
        with pytest.raises(ValueError):
            pool.struct()
        setattr(pool, name, kept)
    pool.a = torch.zeros(2, 3, 10)
    assert pool.struct()._obj.k == 10


def test_a_scale_takes_no_gradient():
    with pytest.raises(ValueError, match="scale"):
        adapters.Adapters(torch.zeros(2, 4, 8), torch.zeros(2, 4, 8), torch.ones(2, requires_grad=True))
    pool = adapters.Adapters(torch.zeros(2, 4, 8), torch.zeros(2, 4, 8))
    with pytest.raises(ValueError, match="out"):
        adapters.add(torch.zeros(1, 8), torch.zeros(1, 8), pool, torch.zeros(1, dtype=torch.int64), out=torch.zeros(1, 8, requires_grad=True))
