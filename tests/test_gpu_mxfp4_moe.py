"""Routed experts in the microscaled four-bit format against the FP64 oracle. Tolerances are the oracle's: what FP32 sums can move, and
the roundings of the results."""
import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu
PAIR_ROUNDING_ROWS = 1024  # from this many rows a summed call keeps its pairs in BF16


def _stack(e, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(e, n, k, generator=g) / k ** 0.5
    return om.quantize(w)


def _experts(e, hidden, inter, gated, seed, hidden_out=None, base=0):
    from hibana_amd.kernels import mxfp4_moe
    fc1, fc2 = _stack(e, 2 * inter if gated else inter, hidden, seed), _stack(e, hidden_out or hidden, inter, seed + 1)
    return mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*fc1, *fc2)), base=base), fc1, fc2


def _call(m, e, k, hidden, seed, skew=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, hidden, generator=g).bfloat16()
    logits = torch.randn(m, e, generator=g) + (3.0 * torch.arange(e).flip(0) / e if skew else 0.0)
    w, ids = torch.topk(logits, k, dim=-1)
    return x, ids.to(torch.int32), torch.softmax(w, -1)


def _check(got, want, off, rounding=2.0 ** -8):
    far = (got.double().cpu() - want).abs()
    bound = off * 1.001 + rounding * 1.01 * (want.abs() + off) + 1e-30
    assert bool((far <= bound).all()), float((far / bound).max())


SIZES = [  # rows, experts, top k, hidden, inter, gated
    (1, 8, 2, 256, 128, True), (1, 512, 10, 2048, 512, True), (1, 3, 3, 32, 32, True), (2, 16, 5, 96, 160, False), (4, 64, 22, 1024, 2688, False), (5, 7, 7, 544, 96, True),
    (13, 33, 4, 288, 224, True), (32, 100, 10, 512, 256, True), (40, 4, 2, 128, 64, False), (65, 24, 6, 256, 480, True), (150, 16, 3, 640, 128, False), (333, 12, 8, 256, 96, True), (1100, 9, 4, 96, 64, True), (512, 100, 1, 64, 96, False),
    (3, 9, 5, 2080, 2080, False), (2, 9, 6, 2144, 2080, True), (70, 6, 3, 1280, 1120, True), (30, 40, 4, 2080, 1056, False), (25, 90, 4, 1184, 96, True), (100, 4, 2, 1056, 1184, False),
    (60, 3, 2, 640, 64, True), (20, 50, 4, 800, 64, True),
    (700, 4, 3, 544, 352, True), (400, 3, 2, 1120, 1056, False), (129, 1, 1, 32, 32, True), (1500, 5, 4, 96, 2080, True), (260, 2, 2, 64, 96, False)]


@pytest.mark.parametrize("m, e, k, hidden, inter, gated", SIZES)
def test_routed_sum_and_pairs(m, e, k, hidden, inter, gated):
    from hibana_amd.kernels import mxfp4_moe
    ex, fc1, fc2 = _experts(e, hidden, inter, gated, 10 * m + e)
    x, ids, w = _call(m, e, k, hidden, m + e, skew=m % 2 == 0)
    args = (ex, x.cuda(), ids.cuda(), w.cuda())
    got = mxfp4_moe.mxfp4_moe(*args)
    assert got.dtype == torch.bfloat16 and got.shape == (m, hidden)
    y, off = om.moe_pairs(x, ids, fc1, fc2)
    want, far = om.moe(x, ids, w, fc1, fc2)
    if m >= PAIR_ROUNDING_ROWS:
        far = far + 2.0 ** -8 * ((y.abs() + off) * w.double()[..., None]).sum(1)
    _check(got, want, far)
    pairs = mxfp4_moe.mxfp4_moe(*args, pairs=True)
    assert pairs.dtype == torch.float32
    _check(pairs, y.flatten(0, 1), off.flatten(0, 1), 2.0 ** -24)
    _check(mxfp4_moe.mxfp4_moe(*args, pairs=True, pairs_bf16=True), y.flatten(0, 1), off.flatten(0, 1))
    assert torch.equal(got, mxfp4_moe.mxfp4_moe(*args))  # repeatable


@pytest.mark.parametrize("m", [1, 6, 20, 130])
def test_ids_outside_the_range_rows_of_none_and_repeats(m):
    """A range of the experts, rows that name none of them (their sums are zero), an expert named twice by a row."""
    from hibana_amd.kernels import mxfp4_moe
    ex, fc1, fc2 = _experts(6, 256, 96, True, 3, base=4)
    x, ids, w = _call(m, 16, 5, 256, m)
    ids[0] = torch.tensor([16, 0, 3, 10, -1])  # none of 4 .. 9
    if m > 2:
        ids[1] = torch.tensor([5, 5, 9, 5, 0])
        w[2] = 0.0
        x[3] = 0.0
    got = mxfp4_moe.mxfp4_moe(ex, x.cuda(), ids.cuda(), w.cuda())
    _check(got, *om.moe(x, ids, w, fc1, fc2, base=4))
    assert not got[0].any()
    nothing = mxfp4_moe.mxfp4_moe(ex, x.cuda(), torch.full_like(ids, 100).cuda(), w.cuda())
    assert nothing.shape == (m, 256) and not nothing.any()


@pytest.mark.parametrize("m", [1, 9, 40, 300, 1200])
def test_nothing_of_a_pair_outside_the_range_is_read(m):
    """Its weight and its place among the pairs' outputs may hold anything, a NaN too; memory the call is given as scratch as well."""
    from hibana_amd.kernels import mxfp4_moe
    ex, fc1, fc2 = _experts(5, 128, 96, m != 40, 21, base=2)
    x, ids, w = _call(m, 10, 4, 128, m)
    inside = (ids >= 2) & (ids < 7)
    clean = torch.where(inside, w, torch.zeros_like(w))
    args = x.cuda(), ids.cuda(), torch.where(inside, w, torch.full_like(w, float("nan"))).cuda()
    mxfp4_moe.tile(ex)
    poison = torch.full((1 << 24,), float("nan"), device="cuda")
    del poison  # what is allocated next lies in it
    got = mxfp4_moe.mxfp4_moe(ex, *args)
    assert bool(torch.isfinite(got).all())
    assert torch.equal(got, mxfp4_moe.mxfp4_moe(ex, args[0], args[1], clean.cuda()))
    want, off = om.moe(x, ids, clean, fc1, fc2, base=2)
    if m >= PAIR_ROUNDING_ROWS:
        y, far = om.moe_pairs(x, ids, fc1, fc2, base=2)
        off = off + 2.0 ** -8 * ((y.abs() + far) * clean.double()[..., None]).sum(1)
    _check(got, want, off)


def test_every_row_on_one_expert_and_a_row_that_is_not_finite():
    from hibana_amd.kernels import mxfp4_moe
    ex, fc1, fc2 = _experts(5, 128, 64, True, 8)
    for m in (3, 47, 200):
        x, ids, w = _call(m, 5, 2, 128, m)
        ids[:, 0], ids[:, 1] = 2, 4
        x[1, 9] = float("nan")
        got = mxfp4_moe.mxfp4_moe(ex, x.cuda(), ids.cuda(), w.cuda())
        assert bool(got[1].isnan().all())
        keep = [i for i in range(m) if i != 1]
        want, off = om.moe(x[keep], ids[keep], w[keep], fc1, fc2)
        _check(got[keep], want, off)


def test_outputs_narrower_or_wider_than_the_input_and_types_of_ids():
    from hibana_amd.kernels import mxfp4_moe
    for m, out in ((1, 8), (9, 520), (70, 96)):
        ex, fc1, fc2 = _experts(9, 160, 64, m != 9, out, hidden_out=out)
        x, ids, w = _call(m, 9, 3, 160, out)
        got = mxfp4_moe.mxfp4_moe(ex, x.cuda(), ids.long().cuda(), w.bfloat16().cuda())
        _check(got, *om.moe(x, ids, w.bfloat16().float(), fc1, fc2))


def test_layout_released_and_nothing_to_do():
    from hibana_amd.kernels import mxfp4_moe
    for gated in (True, False):
        ex, fc1, fc2 = _experts(4, 96, 32, gated, 2)
        mxfp4_moe.tile(ex, release=True)
        assert ex.fc1_codes is None and ex.gated == gated and ex.bytes == 4 * ((2 if gated else 1) * 32 * 96 + 96 * 32) * 17 // 32
        assert all(torch.equal(a.cpu(), b) for fc, want in ((True, fc1), (False, fc2)) for a, b in zip(ex.held(fc), want))
        empty = mxfp4_moe.mxfp4_moe(ex, torch.empty(0, 96, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, 3, device="cuda"))
        assert empty.shape == (0, 96)
        none = mxfp4_moe.mxfp4_moe(ex, torch.ones(2, 96, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 0, dtype=torch.int32, device="cuda"), torch.empty(2, 0, device="cuda"))
        assert none.shape == (2, 96) and not none.any()


@pytest.mark.parametrize("m", [1, 12, 90])
def test_streams_and_graphs(m):
    """The call on another stream, and two captured graphs of it replayed side by side with eager work in between."""
    from hibana_amd.kernels import mxfp4_moe
    ex, _, _ = _experts(20, 256, 128, True, m)
    mxfp4_moe.tile(ex)

    def inputs(seed):
        x, ids, w = _call(m, 20, 4, 256, seed)
        return x.cuda(), ids.cuda(), w.cuda()

    a, b = inputs(1), inputs(2)
    want_a, want_b = mxfp4_moe.mxfp4_moe(ex, *a), mxfp4_moe.mxfp4_moe(ex, *b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = mxfp4_moe.mxfp4_moe(ex, *a)
    here = mxfp4_moe.mxfp4_moe(ex, *b)  # in flight together
    torch.cuda.synchronize()
    assert torch.equal(there, want_a) and torch.equal(here, want_b)
    held = [[t.clone() for t in a], [t.clone() for t in b]]
    graphs, outs = [], []
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(mxfp4_moe.mxfp4_moe(ex, *h))
        graphs.append(graph)
    for seed in range(3):
        fresh = [inputs(10 + seed), inputs(20 + seed)]
        for h, f in zip(held, fresh):
            for t, v in zip(h, f):
                t.copy_(v)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        want = [mxfp4_moe.mxfp4_moe(ex, *f) for f in fresh]
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
