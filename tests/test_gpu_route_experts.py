"""Routing to experts (`ops.route_experts`) and its gradient (`ops.route_experts_grad`) against the rule in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import route_experts as oracle

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SHAPES = [  # m, e, k, groups, kept
    (1, 1, 1, 1, 1),
    (1, 512, 10, 1, 1),
    (3, 8, 8, 1, 1),
    (7, 60, 4, 1, 1),
    (65, 63, 63, 1, 1),
    (130, 256, 8, 8, 4),
    (50, 160, 6, 8, 3),
    (33, 192, 8, 12, 5),     # groups that do not fill the wavefront
    (20, 64, 5, 64, 9),      # of one expert
    (40, 66, 7, 33, 7),      # of two, a lane each
    (31, 96, 12, 3, 1),
    (100, 512, 22, 1, 1),
    (64, 513, 9, 1, 1),
    (29, 1024, 32, 16, 8),
    (23, 1000, 40, 2, 2),
    (9, 1024, 63, 1, 1),
]


def make(m, e, dtype, seed, masked=0.2, bias=0.0):
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(m, e, generator=g)
    logits.masked_fill_(torch.rand(m, e, generator=g) < masked, -torch.inf)
    if m > 2:
        logits[m // 2] = -torch.inf  # a row that a mask leaves nothing of
        logits[m // 2 - 1, 1:] = -torch.inf
    b = bias * torch.randn(e, generator=g) if bias else None
    return logits.to(dtype), b


def check(logits, k, scoring, bias, groups, kept, renormalize, scale, slots=None, steps=1):
    from hibana_amd.kernels import ops
    ids, weights = ops.route_experts(logits.cuda(), k, scoring, bias=None if bias is None else bias.cuda(), groups=groups, kept=kept, renormalize=renormalize, scale=scale,
                                     slots=None if slots is None else slots.cuda(), steps=steps)
    padded = None if slots is None else slots.repeat_interleave(steps).eq(0).numpy()
    l = logits.double().numpy()
    want = oracle.choose(l, k, scoring, None if bias is None else bias.double().numpy(), groups, kept, padded)
    assert ids.dtype == torch.int32 and np.array_equal(ids.cpu().numpy(), want)
    w = oracle.weights(l, want, scoring, renormalize, scale)
    # A score: the exponential's argument l - max is rounded (2^-24 of it, some 20 at most where the score is not below 2^-28 of the largest: there the absolute
    # bound holds), the exponential 2^-23, a sum of 16 + 6 roundings, a division and a product: under 2^-18 in all
    assert np.all(np.abs(weights.cpu().double().numpy() - w) <= 2.0 ** -18 * np.abs(w) + 2.0 ** -45)
    return ids, weights


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("m,e,k,groups,kept", SHAPES)
def test_route(m, e, k, groups, kept, scoring, kind):
    for seed, (bias, renormalize, masked) in enumerate([(0.0, True, 0.2), (0.1, True, 0.0), (0.02, False, 0.3), (0.0, False, 0.0)]):
        logits, b = make(m, e, TYPES[kind], seed, masked, bias)
        check(logits, k, scoring, b, groups, kept, renormalize, 2.5 if seed % 2 else 1.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3)])
def test_equal_and_nearly_equal_choices(groups, kept, scoring):
    """Ties go to the lower expert; scores plus biases that FP32 does not tell apart (or tells apart the wrong way) are told apart."""
    g = torch.Generator().manual_seed(3)
    m, e, k = 200, 256, 9
    few = torch.randint(0, 4, (m, e), generator=g).float() / 8
    check(few, k, scoring, None, groups, kept, True, 1.0)
    check(few.bfloat16(), k, scoring, torch.zeros(e), groups, kept, True, 1.0)
    bias = (torch.randint(0, 3, (e,), generator=g).float() - 1) / 16
    check(few, k, scoring, bias, groups, kept, False, 1.0)
    # biases that even the scores of row 0 out but for their roundings
    logits = torch.randn(1, e, generator=g).expand(m, e).contiguous()
    logits[1:] += 1e-7 * torch.randn(m - 1, e, generator=g)
    near = (1.0 - torch.from_numpy(oracle.scores(logits[:1].double().numpy(), scoring))[0]).float()
    check(logits, k, scoring, near, groups, kept, True, 1.0)
    both = torch.zeros(4, e)
    both[0] = torch.where(torch.arange(e) % 2 == 0, 0.0, -0.0)  # both zeros are one value
    check(both, k, scoring, None, groups, kept, True, 1.0)
    check(both, k, scoring, torch.where(torch.arange(e) % 2 == 0, 0.0, -0.0), groups, kept, True, 1.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_far_logits(scoring):
    """Scores that FP32 does not hold renormalize all the same, in the order of the logits."""
    g = torch.Generator().manual_seed(5)
    for shift in (-300.0, 300.0, 0.0):
        logits = shift + 30 * torch.randn(40, 100, generator=g)
        check(logits, 6, scoring, None, 1, 1, True, 1.0)
    check(-torch.rand(10, 100, generator=g) * 3e38, 6, scoring, None, 1, 1, True, 1.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_what_is_not_a_number(groups, kept, bias, scoring):
    from hibana_amd.kernels import ops
    g = torch.Generator().manual_seed(6)
    m, e, k = 12, 64, 5
    logits = torch.randn(m, e, generator=g)
    logits[1, 7] = torch.nan
    logits[2] = torch.nan
    logits[3, 9] = torch.inf
    logits[4, :62] = -torch.inf
    b = 0.1 * torch.randn(e, generator=g) if bias else None
    if bias:
        b[3], b[4], b[5] = -torch.inf, torch.nan, torch.inf
    ids, weights = ops.route_experts(logits.cuda(), k, scoring, bias=None if b is None else b.cuda(), groups=groups, kept=kept)
    ids, weights = ids.cpu().numpy(), weights.cpu()
    l = logits.double().numpy()
    want = oracle.choose(l, k, scoring, None if b is None else b.double().numpy(), groups, kept)
    assert np.array_equal(ids, want)
    real = torch.from_numpy(want < e)
    assert weights[1][real[1]].isnan().all() and (ids[2] == e).all() and not weights[2].any()
    assert weights[3][real[3]].isnan().all() == (scoring == "softmax")
    for r in [0, *range(4, m)]:
        assert weights[r].isfinite().all() and abs(weights[r].sum().item() - 1.0) < 1e-5 and not weights[r][~real[r]].any(), r


def test_rows_as_they_come():
    """A stride, odd addresses, padded requests of several rows, int64 and bool slots, rows of one expert."""
    from hibana_amd.kernels import ops
    g = torch.Generator().manual_seed(7)
    for dtype in TYPES.values():
        wide = torch.randn(24, 101, generator=g).to(dtype).cuda()
        part = wide[:, 3:98]
        want = ops.route_experts(part.contiguous(), 7, "sigmoid")
        for got, w in zip(ops.route_experts(part, 7, "sigmoid"), want):
            assert torch.equal(got, w)
        dw = torch.randn(24, 7, device="cuda")
        assert torch.equal(ops.route_experts_grad(dw, part, want[0], "sigmoid"), ops.route_experts_grad(dw, part.contiguous(), want[0], "sigmoid"))
        assert torch.equal(ops.route_experts(part.t().contiguous().t(), 7, "sigmoid")[1], want[1])
    logits, _ = make(24, 95, torch.float32, 8)
    slots = torch.tensor([1, 0, 3, 0, 1, 1, 0, 9], dtype=torch.int32)
    ids, weights = check(logits, 7, "softmax", None, 1, 1, True, 1.0, slots, 3)
    again = ops.route_experts(logits.cuda(), 7, slots=slots.long().cuda(), steps=3)
    assert torch.equal(again[0], ids) and torch.equal(ops.route_experts(logits.cuda(), 7, slots=(slots != 0).cuda(), steps=3)[0], ids)
    ids, weights = ops.route_experts(torch.randn(0, 20, device="cuda"), 3)
    assert ids.shape == weights.shape == (0, 3)
    assert ops.route_experts_grad(weights, torch.randn(0, 20, device="cuda"), ids).shape == (0, 20)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("m,e,k,groups,kept", SHAPES)
def test_gradient(m, e, k, groups, kept, renormalize, scoring, kind):
    from hibana_amd.kernels import ops
    logits, _ = make(m, e, TYPES[kind], 9)
    ids = torch.from_numpy(oracle.choose(logits.double().numpy(), k, scoring, None, groups, kept)).int()
    dw = torch.randn(m, k, generator=torch.Generator().manual_seed(10))
    if m > 5:
        ids[3, 0] = -4                     # ids that name no expert add nothing
        ids[4, -1] = ids[4, 0]             # one expert twice
    got = ops.route_experts_grad(dw.cuda(), logits.cuda(), ids.cuda(), scoring, renormalize=renormalize, scale=1.5).cpu().double().numpy()
    l = logits.double().numpy()
    want = oracle.grad(dw.numpy(), l, ids.numpy(), scoring, renormalize, 1.5)
    # scores as in `check` (2^-18); the difference dw - sum of dw w cancels: of the size of the largest |dw|; one rounding to the type
    real = (ids.numpy() >= 0) & (ids.numpy() < e)
    top = 1.5 * np.where(real, np.abs(dw.numpy()), 0).max(1, keepdims=True)
    score = np.abs(oracle.grad(np.ones((m, k)), l, ids.numpy(), "sigmoid", False, 1.0)) if scoring == "sigmoid" else oracle.scores(l, scoring)
    if renormalize:
        score = np.zeros((m, e))
        for r in range(m):
            np.add.at(score[r], np.where(real, ids.numpy(), 0)[r], np.where(real, oracle.weights(l, np.where(real, ids.numpy(), e), scoring, True, 1.0), 0.0)[r])
    bound = 2.0 ** -16 * score * top * (1 + k) + torch.finfo(TYPES[kind]).eps / 2 * np.abs(want) + {"f16": 2.0 ** -25, "bf16": 2.0 ** -45, "f32": 2.0 ** -45}[kind]
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_by_differences(renormalize, scoring):
    """Central differences of the weights over the logits, at ids that do not change: f's third derivative is below 1 in size for scores below 1, so h^2 / 6 of
    k |dw|, and 2^-18 of the weights over 2 h."""
    from hibana_amd.kernels import ops
    g = torch.Generator().manual_seed(11)
    m, e, k, h = 30, 40, 4, 2.0 ** -5
    logits = torch.arange(e).float()[None].expand(m, e)[:, torch.randperm(e, generator=g)] * 0.15  # far enough apart
    dw = torch.randn(m, k, generator=g)
    step = torch.sign(torch.randn(m, e, generator=g))
    ids, _ = ops.route_experts(logits.cuda(), k, scoring, renormalize=renormalize)
    ends = []
    for s in (h, -h):
        i, w = ops.route_experts((logits + s * step).cuda(), k, scoring, renormalize=renormalize)
        assert torch.equal(i, ids)
        ends.append((w.cpu().double() * dw).sum(1))
    got = ops.route_experts_grad(dw.cuda(), logits.cuda(), ids, scoring, renormalize=renormalize).cpu().double()
    off = ((ends[0] - ends[1]) / (2 * h) - (got * step).sum(1)).abs()
    assert (off <= dw.abs().sum(1) * (k * h * h / 6 * 4 + 2.0 ** -18 / h)).all()


def test_autograd_and_captures():
    from hibana_amd.kernels import ops
    logits, b = make(50, 96, torch.bfloat16, 12, bias=0.1)
    logits, b = logits.cuda(), b.cuda()
    rule = dict(bias=b, groups=4, kept=2, renormalize=True, scale=2.0)
    leaf = logits.clone().requires_grad_()
    ids, weights = ops.route_experts(leaf, 6, "sigmoid", **rule)
    want = ops.route_experts(logits, 6, "sigmoid", **rule)
    assert torch.equal(ids, want[0]) and torch.equal(weights.detach(), want[1]) and not ids.requires_grad
    dw = torch.randn_like(weights)
    weights.backward(dw)
    assert torch.equal(leaf.grad, ops.route_experts_grad(dw, logits, ids, "sigmoid", scale=2.0))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.route_experts(logits, 6, "sigmoid", **rule)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            ops.route_experts(leaf, 6, "sigmoid", **rule)
        got = ops.route_experts(logits, 6, "sigmoid", **rule)
        grad = ops.route_experts_grad(dw, logits, got[0], "sigmoid", scale=2.0)
    for i in range(4):
        logits.copy_(torch.randn(50, 96)), dw.copy_(torch.randn(50, 6)), b.copy_(0.1 * torch.randn(96))
        graph.replay()
        want = ops.route_experts(logits, 6, "sigmoid", **rule)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(grad, ops.route_experts_grad(dw, logits, want[0], "sigmoid", scale=2.0)), i


def test_the_rules_that_the_other_entry_points_have():
    """Without bias, groups and mask: `route_topk`'s choice and weights."""
    from hibana_amd.kernels import ops
    logits = torch.randn(100, 432, generator=torch.Generator().manual_seed(13)).cuda()
    ids, weights = ops.route_topk(logits, 9)
    got = ops.route_experts(logits, 9)
    assert torch.equal(got[0], ids)
    torch.testing.assert_close(got[1], weights, rtol=2.0 ** -17, atol=0.0)
