"""Low-rank adapters beside a shared projection (`adapters.add`) and their gradients (`adapters.grads`) against the formula in 64 bits."""
import pytest
import torch

from oracle import adapters as oracle

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def make(m, k, n, rank, count, dtype, seed=0, runs=0, ragged=False, none=False, scaled=True):
    """CPU tensors: y, x, a, b, scale, ranks, index."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    y, x = normal(m, n).to(dtype), normal(m, k).to(dtype)
    a, b = (normal(count, rank, k) / k ** 0.5).to(dtype), (normal(count, rank, n) * 0.3).to(dtype)
    scale = 0.5 + torch.rand(count, generator=g) if scaled else None
    ranks = torch.randint(0 if none else 1, rank + 1, (count,), generator=g, dtype=torch.int32) if ragged else None
    low = -1 if none else 0
    if runs:
        cuts = sorted(torch.randint(0, m + 1, (runs - 1,), generator=g).tolist())
        owner = torch.randint(low, count, (runs,), generator=g)
        index = torch.cat([owner[i:i + 1].expand(hi - lo) for i, (lo, hi) in enumerate(zip([0, *cuts], [*cuts, m]))])
    else:
        index = torch.randint(low, count, (m,), generator=g)
    return y, x, a, b, scale, ranks, index.to(torch.int32)


def pool_of(a, b, scale, ranks):
    from hibana_amd.kernels import adapters
    return adapters.Adapters(*(None if t is None else t.cuda() for t in (a, b, scale, ranks)))


def within(got, want, bound, what):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst} times the bound"


SIZES = [  # m, k, n, rank, adapters, runs, ragged, none
    (1, 64, 64, 16, 1, 0, False, False),
    (1, 5120, 640, 16, 8, 0, False, False),
    (2, 1, 1, 1, 1, 0, False, False),
    (5, 7, 1025, 3, 2, 0, False, True),
    (16, 129, 513, 33, 3, 0, True, True),
    (17, 1000, 127, 16, 1, 0, False, False),   # two tiles of one adapter
    (64, 640, 2049, 64, 32, 0, True, True),
    (77, 2560, 255, 24, 16, 5, False, False),
    (255, 65, 100, 8, 300, 0, False, True),
    (256, 320, 300, 17, 2, 0, False, True),    # the last size that finds its tiles itself
    (257, 320, 300, 17, 2, 0, False, True),    # the first with a plan
    (300, 96, 1024, 40, 1, 1, False, False),
    (700, 1111, 333, 100, 5, 9, True, True),
    (1000, 64, 72, 4, 4096, 0, False, True),   # a pool as large as it gets, most of it unused
    (513, 72, 65, 256, 3, 4, False, False),
    (2047, 136, 264, 16, 3, 7, False, True),
    (2049, 200, 520, 48, 7, 30, True, True),
    (4100, 130, 70, 32, 2, 0, False, False),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,k,n,rank,count,runs,ragged,none", SIZES)
def test_add(m, k, n, rank, count, runs, ragged, none, kind):
    from hibana_amd.kernels import adapters
    case = make(m, k, n, rank, count, TYPES[kind], seed=m + n, runs=runs, ragged=ragged, none=none)
    y, x, a, b, scale, ranks, index = case
    got = adapters.add(y.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda())
    within(got, oracle.add(*case), oracle.add_bound(*case), "out")
    free = index < 0
    if ranks is not None:
        free |= ranks[index.clamp(min=0).long()] == 0
    assert torch.equal(got.cpu()[free], y[free])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,k,n,rank,count,runs,ragged,none", SIZES)
def test_grads(m, k, n, rank, count, runs, ragged, none, kind):
    from hibana_amd.kernels import adapters
    case = make(m, k, n, rank, count, TYPES[kind], seed=m + n + 1, runs=runs, ragged=ragged, none=none)
    dy, x, a, b, scale, ranks, index = case
    got = adapters.grads(dy.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda())
    assert [t.dtype for t in got] == [x.dtype, torch.float32, torch.float32]
    for name, g, w, bound in zip(("dx", "da", "db"), got, oracle.grads(*case), oracle.grads_bound(*case)):
        within(g, w, bound, name)
        assert not g.cpu()[w == 0].any()  # (rows without an adapter, adapters without a row, rows behind a rank: zeros, whatever else)


def test_gradients_by_differences():
    """(f(p + h) - f(p - h)) / 2 h of f = the sum of `add`'s result times fixed weights, in 32 bits: f is linear in x, in a and in b, so the difference is the
    gradient but for rounding: f is a sum of m n terms of FP32 results, each off by 2^-23 of about its size, over 2 h."""
    from hibana_amd.kernels import adapters
    dy, x, a, b, scale, ranks, index = make(33, 40, 50, 6, 3, torch.float32, seed=4, ragged=True, none=True)
    y = torch.zeros_like(dy).cuda()
    dx, da, db = (t.cpu().double() for t in adapters.grads(dy.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda()))
    g = torch.Generator().manual_seed(5)

    def f(x, a, b):
        return (adapters.add(y, x.cuda(), pool_of(a, b, scale, ranks), index.cuda()).cpu().double() * dy.double()).sum().item()
    for name, at in (("x", 0), ("a", 1), ("b", 2)):
        base = [x, a, b]
        step = torch.sign(torch.randn(base[at].shape, generator=g))
        h = 0.5
        ends = []
        for sign in (h, -h):
            moved = list(base)
            moved[at] = base[at] + sign * step
            ends.append(f(*moved))
        want = ((dx, da, db)[at] * step.double()).sum().item()
        size = adapters.add(y, x.abs().cuda() + h, pool_of(a.abs() + h, b.abs() + h, scale, ranks), index.cuda()).cpu().double().mul(dy.abs().double()).sum().item()
        assert abs((ends[0] - ends[1]) / (2 * h) - want) <= 2 * (40 + 12 + 16) * 2.0 ** -23 * size, name


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m", [40, 400])
def test_autograd_gives_the_same_gradients(m, kind):
    from hibana_amd.kernels import adapters
    case = make(m, 96, 80, 8, 3, TYPES[kind], seed=6, none=True)
    dy, x, a, b, scale, ranks, index = (None if t is None else t.cuda() for t in case)
    y = torch.randn_like(dy).requires_grad_()
    xg = x.clone().requires_grad_()
    pool = adapters.Adapters(torch.nn.Parameter(a), torch.nn.Parameter(b), scale)
    out = adapters.add(y, xg, pool, index)
    assert torch.equal(out.detach(), adapters.add(y.detach(), x, adapters.Adapters(a, b, scale), index))
    out.backward(dy)
    dx, da, db = adapters.grads(dy, x, adapters.Adapters(a, b, scale), index)
    assert torch.equal(xg.grad, dx) and torch.equal(pool.a.grad, da.to(a.dtype)) and torch.equal(pool.b.grad, db.to(b.dtype)) and torch.equal(y.grad, dy)
    with torch.no_grad():
        adapters.add(y, xg, pool, index, out=y.detach())
    with pytest.raises(ValueError):
        adapters.add(y, xg, pool, index, out=torch.empty_like(dy))


@pytest.mark.parametrize("m", [50, 300])
def test_rows_as_they_come(m):
    """Strides, odd addresses, int64 indexes that 32 bits do not hold, `out` of its own stride and y itself."""
    from hibana_amd.kernels import adapters
    y, x, a, b, scale, ranks, index = make(m, 95, 131, 12, 4, torch.bfloat16, seed=8, none=True)
    pool = pool_of(a, b, scale, ranks)
    want = adapters.add(y.cuda(), x.cuda(), pool, index.cuda())
    wide_x = torch.randn(m, 200, device="cuda").bfloat16()
    wide_y = torch.randn(m, 301, device="cuda").bfloat16()
    wide_x[:, 3:98], wide_y[:, 5:136] = x.cuda(), y.cuda()
    far = torch.where(index < 0, 2 ** 32 + 1, index.long()).cuda()
    out = torch.full((m, 200), 7.0, device="cuda").bfloat16()
    got = adapters.add(wide_y[:, 5:136], wide_x[:, 3:98], pool, far, out=out[:, 9:140])
    assert got.data_ptr() == out[:, 9:].data_ptr() and torch.equal(got, want)
    assert (out[:, :9] == 7).all() and (out[:, 140:] == 7).all()
    before = wide_y.clone()
    adapters.add(wide_y[:, 5:136], wide_x[:, 3:98], pool, far, out=wide_y[:, 5:136])
    assert torch.equal(wide_y[:, 5:136], want) and torch.equal(wide_y[:, :5], before[:, :5]) and torch.equal(wide_y[:, 136:], before[:, 136:])
    columns = x.cuda().t().contiguous().t()  # rows not contiguous: copied
    assert torch.equal(adapters.add(y.cuda(), columns, pool, torch.stack((index, index), 1).cuda()[:, 0]), want)
    spread = x[:1].cuda().expand(m, 95)
    assert torch.equal(adapters.add(y.cuda(), spread, pool, index.cuda()), adapters.add(y.cuda(), spread.contiguous(), pool, index.cuda()))
    dy = y
    first = adapters.grads(dy.cuda(), x.cuda(), pool, index.cuda())
    wide_y[:, 5:136] = dy.cuda()
    for u, v in zip(first, adapters.grads(wide_y[:, 5:136], wide_x[:, 3:98], pool, far)):
        assert torch.equal(u, v)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m", [200, 600])
def test_a_row_is_its_own(m, kind):
    """Rows in another order give the same rows; NaN and infinities in some rows, in y, and behind an adapter's rank, reach no other row."""
    from hibana_amd.kernels import adapters
    y, x, a, b, scale, ranks, index = make(m, 100, 90, 20, 5, TYPES[kind], seed=9, ragged=True, none=True)
    behind = torch.arange(20)[None, :, None] >= ranks[:, None, None]
    pool = pool_of(a.masked_fill(behind, float("nan")), b.masked_fill(behind, float("inf")), scale, ranks)
    want = adapters.add(y.cuda(), x.cuda(), pool, index.cuda())
    within(want, oracle.add(y, x, a, b, scale, ranks, index), oracle.add_bound(y, x, a, b, scale, ranks, index), "out")
    turn = torch.randperm(m, generator=torch.Generator().manual_seed(1))
    assert torch.equal(adapters.add(y[turn].cuda(), x[turn].cuda(), pool, index[turn].cuda()).cpu(), want.cpu()[turn])
    bad = torch.zeros(m, dtype=torch.bool)
    bad[::7] = True
    x2, y2 = x.clone(), y.clone()
    x2[::14, 3], x2[7::14, 50] = float("nan"), float("inf")
    y2[::7, 11] = float("-inf")
    got = adapters.add(y2.cuda(), x2.cuda(), pool, index.cuda())
    assert torch.equal(got.cpu()[~bad], want.cpu()[~bad])
    free = (index < 0) | (ranks[index.clamp(min=0).long()] == 0)
    assert torch.equal(got.cpu()[free], y2[free])
    with_nan = bad & ~free & (torch.arange(m) % 14 == 0)
    assert got.cpu()[with_nan].isnan().any(1).all()
    dx, da, db = adapters.grads(y.cuda(), x.cuda(), pool, index.cuda())
    for g, w, bound in zip((dx, da, db), oracle.grads(y, x, a, b, scale, ranks, index), oracle.grads_bound(y, x, a, b, scale, ranks, index)):
        within(g, w, bound, "gradient")
    dx2, da2, db2 = adapters.grads(y.cuda(), x2.cuda(), pool, index.cuda())
    assert torch.equal(dx2, dx) and da2.isnan().any()  # (dx is of dy alone)


@pytest.mark.parametrize("m", [3, 300])
def test_sums_past_the_type(m):
    """FP16: inner sums past 65504 and below its smallest value; BF16 and FP32: far from one."""
    from hibana_amd.kernels import adapters
    for kind, big in (("f16", 2.0 ** 10), ("bf16", 2.0 ** 40), ("f32", 2.0 ** 40)):
        dtype = TYPES[kind]
        for up, down in ((big, 1 / big), (2.0 ** -12, 2.0 ** 8)):
            y, x, a, b, scale, ranks, index = make(m, 512, 70, 9, 2, dtype, seed=10)
            x, a, b = (x.float() * up).to(dtype), (a.float() * 22 * up).to(dtype), (b.float() * down).to(dtype)
            scale = torch.full((2,), 1 / up)
            case = (y, x, a, b, scale, ranks, index)
            within(adapters.add(y.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda()), oracle.add(*case), oracle.add_bound(*case), f"{kind} {up}")
            dy = (y.float() * 1e-3).to(dtype)
            case = (dy, x, a, b, scale, ranks, index)
            if oracle.grads(*case)[0].abs().max() < torch.finfo(dtype).max:
                for g, w, bound in zip(adapters.grads(dy.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda()), oracle.grads(*case), oracle.grads_bound(*case)):
                    within(g, w, bound, f"{kind} {up}")


@pytest.mark.parametrize("m", [0, 1])
def test_no_rows_and_one(m):
    from hibana_amd.kernels import adapters
    y, x, a, b, scale, ranks, index = make(1, 30, 20, 4, 2, torch.float32)
    pool = pool_of(a, b, None, None)
    y, x, index = y[:m].cuda(), x[:m].cuda(), index[:m].cuda()
    assert adapters.add(y, x, pool, index).shape == (m, 20)
    dx, da, db = adapters.grads(y, x, pool, index)
    assert dx.shape == (m, 30) and da.shape == a.shape and db.shape == b.shape and (m or not (da.any() or db.any()))
    if m:
        assert torch.equal(adapters.add(y, x, pool, torch.full((1,), 2, device="cuda")), y)
        assert not any(t.any() for t in adapters.grads(y, x, pool, torch.full((1,), -5, device="cuda")))


@pytest.mark.parametrize("m", [40, 700])
def test_captured_and_replayed(m):
    """`add` and `grads` in a graph, replayed over new inputs, new indexes and an adapter set anew, between eager calls on another stream."""
    from hibana_amd.kernels import adapters
    y, x, a, b, scale, ranks, index = (None if t is None else t.cuda() for t in make(m, 320, 200, 24, 6, torch.bfloat16, seed=11, ragged=True, none=True))
    pool = adapters.Adapters(a, b, scale, ranks)

    def both():
        return (adapters.add(y, x, pool, index), *adapters.grads(y, x, pool, index))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    with torch.cuda.graph(other):
        again = both()
    for i in range(4):
        x.copy_(torch.randn_like(x)), y.copy_(torch.randn_like(y))
        index.copy_(torch.randint(-1, 6, (m,), device="cuda"))
        pool.set(i, torch.randn(5 + i, 320), torch.randn(200, 5 + i), 0.25)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other.replay()  # two graphs side by side share nothing
            want = both()
        torch.cuda.synchronize()
        for g, h, w in zip(got, again, want):
            assert torch.equal(g, w) and torch.equal(h, w), i


def test_a_recorded_gradient_is_refused_in_a_capture():
    from hibana_amd.kernels import adapters
    y, x, a, b, scale, ranks, index = (None if t is None else t.cuda() for t in make(4, 32, 32, 4, 2, torch.float32))
    pool = adapters.Adapters(torch.nn.Parameter(a), torch.nn.Parameter(b))
    with torch.no_grad():
        adapters.add(y, x, pool, index)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            adapters.add(y, x, pool, index)
        with torch.no_grad():
            out = adapters.add(y, x, pool, index)
    graph.replay()
    with torch.no_grad():
        assert torch.equal(out, adapters.add(y, x, pool, index))


def test_a_pool_of_pairs():
    """Checkpoint pairs of different ranks; an adapter replaced; an optimizer that puts another tensor in a parameter's place."""
    from hibana_amd.kernels import adapters
    g = torch.Generator().manual_seed(12)
    pairs = [(torch.randn(r, 60, generator=g), torch.randn(44, r, generator=g), 0.5 + r / 10) for r in (3, 1, 7)]
    pool = adapters.Adapters.from_pairs(pairs, torch.float32)
    assert (pool.adapters, pool.rank, pool.in_features, pool.out_features) == (3, 7, 60, 44) and pool.ranks.tolist() == [3, 1, 7]
    x, y = torch.randn(10, 60, generator=g), torch.randn(10, 44, generator=g)
    index = torch.arange(10) % 4 - 1

    def want():
        out = y.double()
        for r, i in enumerate(index.tolist()):
            if i >= 0:
                out[r] += pairs[i][2] * (pairs[i][1].double() @ (pairs[i][0].double() @ x[r].double()))
        return out
    close = lambda: torch.testing.assert_close(adapters.add(y.cuda(), x.cuda(), pool, index.cuda()).cpu().double(), want(), rtol=1e-5, atol=1e-4)  # noqa: E731
    close()
    pairs[2] = (torch.randn(2, 60, generator=g), torch.randn(44, 2, generator=g), 2.0)
    pool.set(2, *pairs[2])
    close()
    pool.a = pool.a.clone().mul_(2.0)
    pairs = [(p[0] * 2, *p[1:]) for p in pairs]
    close()


@pytest.mark.parametrize("count", [3, 1000])
def test_gradients_of_several_units_of_rows(count):
    """Adapters of many rows, of one and of none in a call, in a small pool and among many: partial sums are those of the adapters that have them."""
    from hibana_amd.kernels import adapters
    m, k, n, rank = 3000, 70, 40, 5
    y, x, a, b, scale, ranks, _ = make(m, k, n, rank, count, torch.bfloat16, seed=30)
    index = torch.full((m,), count - 1, dtype=torch.int32)
    index[::3], index[5], index[6] = 0, 1, -1
    case = (y, x, a, b, scale, ranks, index)
    got = adapters.grads(y.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda())
    for name, g, w, bound in zip(("dx", "da", "db"), got, oracle.grads(*case), oracle.grads_bound(*case)):
        within(g, w, bound, name)
    for g, w in zip(adapters.grads(y.cuda(), x.cuda(), pool_of(a, b, scale, ranks), index.cuda()), got):
        assert torch.equal(g, w)  # the same call, the same bits


@pytest.mark.parametrize("kind", TYPES)
def test_results_and_rows_past_the_caches(kind):
    """Results of more than 16 MB, rows of more than 128: the same sums by other loads and stores (the oracle in 64 bits on the GPU). Odd widths."""
    from hibana_amd.kernels import adapters
    m, k, n, rank, count = 2100, 9, 32001 if kind != "f32" else 16003, 3, 2
    g = torch.Generator(device="cuda").manual_seed(31)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    for wide, narrow in ((n, k), (k, n)):
        y, x = normal(m, wide).to(TYPES[kind]), normal(m, narrow).to(TYPES[kind])
        a, b = (normal(count, rank, narrow) / narrow ** 0.5).to(TYPES[kind]), (0.3 * normal(count, rank, wide)).to(TYPES[kind])
        case = (y, x, a, b, torch.tensor([0.5, 2.0], device="cuda"), None, (torch.arange(m, device="cuda") * 3 // m - 1).int())
        pool, index = adapters.Adapters(a, b, case[4]), case[-1]
        off = (adapters.add(y, x, pool, index).double() - oracle.add(*case)).abs()
        assert bool((off <= oracle.add_bound(*case)).all())
        del off
        for got, want, bound in zip(adapters.grads(y, x, pool, index), oracle.grads(*case), oracle.grads_bound(*case)):
            assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("m,count", [(257, 3), (320, 2559), (320, 2560), (4096, 200), (8192, 118), (8192, 119), (8193, 4), (12000, 300), (20000, 4096)])
def test_rows_among_many_adapters(m, count):
    """The grouping of rows by adapter at the sizes where its kernels, their wavefronts and their counters change. Small whole numbers: every sum is exact."""
    from hibana_amd.kernels import adapters
    g = torch.Generator().manual_seed(m + count)
    whole = lambda *s: torch.randint(-1, 2, s, generator=g)  # noqa: E731
    y, x, a, b = whole(m, 16), whole(m, 8), whole(count, 2, 8), whole(count, 2, 16)
    index = torch.randint(-1, count, (m,), generator=g)
    index[m // 2:m // 2 + 200] = count - 1  # a run of one adapter's among them
    of = index.clamp(min=0)
    there = (index >= 0).long()[:, None]
    inner = (x[:, None, :] * a[of]).sum(2) * there
    back = (y[:, None, :] * b[of]).sum(2) * there
    pool = adapters.Adapters(a.bfloat16().cuda(), b.bfloat16().cuda())
    y16, x16, where = y.bfloat16().cuda(), x.bfloat16().cuda(), index.cuda()
    assert torch.equal(adapters.add(y16, x16, pool, where).cpu().long(), y + (inner[:, :, None] * b[of]).sum(1))
    dx, da, db = (t.cpu().long() for t in adapters.grads(y16, x16, pool, where))
    assert torch.equal(dx, (back[:, :, None] * a[of]).sum(1))
    assert torch.equal(da, torch.zeros_like(a).index_add_(0, of, back[:, :, None] * x[:, None, :]))
    assert torch.equal(db, torch.zeros_like(b).index_add_(0, of, inner[:, :, None] * y[:, None, :]))


def test_a_pool_cut_and_put_elsewhere():
    """Fewer adapters at the same addresses, memory of another shape put in a parameter's place, a copy of a pool in use."""
    import copy
    from hibana_amd.kernels import adapters
    y, x, a, b, scale, _, _ = (None if t is None else t.cuda() for t in make(6, 40, 24, 8, 3, torch.float32, seed=40))
    index = torch.arange(6, device="cuda") % 3
    pool = adapters.Adapters(a, b)
    three = adapters.add(y, x, pool, index)
    other = copy.deepcopy(pool)
    other.b.zero_()
    assert torch.equal(adapters.add(y, x, other, index), y) and torch.equal(adapters.add(y, x, pool, index), three)
    pool.a, pool.b = pool.a[:1], pool.b[:1]
    one = adapters.add(y, x, pool, index)
    assert torch.equal(one[index > 0], y[index > 0]) and torch.equal(one[index == 0], three[index == 0])
    pool.a, pool.b = a, b
    pool.a.data, pool.b.data = a.data[:, :4].contiguous(), b.data[:, :4].contiguous()
    assert torch.equal(adapters.add(y, x, pool, index), adapters.add(y, x, adapters.Adapters(a.clone(), b.clone()), index))


def test_rows_past_four_gibibytes():
    """Rows whose bytes begin past 2^32 from the first's. Whole numbers: every sum is exact, dx is its exact value rounded once."""
    from hibana_amd.kernels import adapters
    m, k, n, rank, count = 900_000, 24, 2504, 2, 3
    g = torch.Generator(device="cuda").manual_seed(50)
    whole = lambda *s: torch.randint(-1, 2, s, device="cuda", dtype=torch.int8, generator=g).bfloat16()  # noqa: E731
    y, x, a, b = whole(m, n), whole(m, k), whole(count, rank, k), whole(count, rank, n)
    index = torch.randint(-1, count, (m,), device="cuda", generator=g)
    pool = adapters.Adapters(a, b)
    out = adapters.add(y, x, pool, index)
    dx, da, db = adapters.grads(y, x, pool, index)
    want_a, want_b = torch.zeros(a.shape, device="cuda", dtype=torch.float64), torch.zeros(b.shape, device="cuda", dtype=torch.float64)
    for at in range(0, m, 50_000):
        rows = slice(at, min(at + 50_000, m))
        ys, xs, to, back = y[rows].float(), x[rows].float(), y[rows].float(), torch.zeros(x[rows].shape, device="cuda")
        for i in range(count):
            of = (index[rows] == i).float()[:, None]
            inner, outer = (xs @ a[i].float().t().contiguous()) * of, (ys @ b[i].float().t().contiguous()) * of
            to += inner @ b[i].float()
            back += outer @ a[i].float()
            want_a[i] += (outer.t().contiguous() @ xs).double()
            want_b[i] += (inner.t().contiguous() @ ys).double()
        assert torch.equal(out[rows], to.bfloat16()) and torch.equal(dx[rows], back.bfloat16()), at
    assert torch.equal(da.double(), want_a) and torch.equal(db.double(), want_b)
