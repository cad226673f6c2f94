"""Routing among groups whose experts have biases near the end of FP32's range: masks of the type's lowest value, infinities, sums of two past the range."""
import pytest
import torch

from tests.test_gpu_route_experts import check

pytestmark = pytest.mark.gpu

LOWEST, HIGHEST = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_a_group_of_lowest_values_comes_before_one_of_none(scoring):
    logits = torch.randn(3, 16, generator=torch.Generator().manual_seed(1))
    logits[:, :4] = -torch.inf
    bias = torch.zeros(16)
    bias[4:12] = LOWEST
    ids, _ = check(logits, 6, scoring, bias, 4, 2, True, 1.0)
    assert (ids < 16).all()
    ids, _ = check(logits, 3, scoring, torch.full((16,), LOWEST), 4, 1, True, 1.0)  # every other group's sum is past the range, as far as the empty one's
    assert (ids < 16).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sums_past_the_range_keep_their_order(scoring):
    logits = torch.randn(3, 16, generator=torch.Generator().manual_seed(2))
    bias = torch.zeros(16)
    bias[4:6], bias[8:10], bias[12:14] = 2.0e38, 2.5e38, 3.0e38
    ids, _ = check(logits, 2, scoring, bias, 4, 1, True, 1.0)
    assert (ids >= 12).all()
    check(logits, 4, scoring, bias, 4, 2, False, 1.0)
    check(logits, 4, scoring, -bias, 4, 2, False, 1.0)
    far = torch.tensor([2.5e38, 1e38, 3.2e38, 2e38, 3e38, 0.5e38])  # 3.5e38, 5.2e38, 3.5e38: in FP32 all of them infinite
    ids, _ = check(logits[:, :6], 1, scoring, far, 3, 1, False, 1.0)
    assert (ids == 2).all()
    check(logits[:, :6], 1, scoring, -far, 3, 1, False, 1.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept,e,k", [(4, 2, 64, 7), (8, 3, 512, 9), (16, 5, 32, 6), (3, 1, 96, 8), (1, 1, 100, 12)])
def test_values_from_all_of_the_range(groups, kept, e, k, scoring):
    g = torch.Generator().manual_seed(e + k)
    of = torch.tensor([0.0, 0.0, 0.1, 1.0, -1e9, 1e9, 1e30, -1e30, 1.1e38, -1.1e38, 2e38, -2e38, LOWEST, HIGHEST, torch.inf, -torch.inf])
    for seed in range(12):
        logits = 2 * torch.randn(20, e, generator=g)
        logits.masked_fill_(torch.rand(20, e, generator=g) < 0.3, -torch.inf)
        logits[3] = LOWEST
        logits[4, ::2] = LOWEST
        bias = of[torch.randint(0, len(of) if seed < 6 else len(of) - 2, (e,), generator=g)]
        if seed % 2:  # one value a group: its sums decide
            bias = bias[:groups].repeat_interleave(e // groups)
        check(logits, k, scoring, bias, groups, kept, True, 1.0)
