"""Slots of any type: a row is padded where its request's slot is zero, and nowhere else."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [torch.tensor([2 ** 32, 0, -2 ** 32, 3, 0, 2 ** 40 + 1]), torch.tensor([0.5, 0.0, -0.25, 3.0, -0.0, 1e20]), torch.tensor([True, False, True, True, False, True]),
                                   torch.tensor([1, 0, 255, 7, 0, 9], dtype=torch.uint8), torch.tensor([-1, 0, 1 << 30, 3, 0, -(1 << 31)], dtype=torch.int32)])
def test_padded_rows(slots):
    from hibana_amd.kernels import ops
    logits = torch.randn(12, 20, generator=torch.Generator().manual_seed(0)).cuda()
    assert torch.equal(ops.route_experts(logits, 3, slots=slots.view(2, 3).t().cuda(), steps=2)[0], ops.route_experts(logits, 3, slots=slots.view(2, 3).t().contiguous().cuda(), steps=2)[0])
    whole, padded = ops.route_experts(logits, 3), slots.ne(0).logical_not().repeat_interleave(2).cuda()
    ids, weights = ops.route_experts(logits, 3, slots=slots.cuda(), steps=2)
    assert torch.equal(ids, whole[0].masked_fill(padded[:, None], 20)) and torch.equal(weights, whole[1].masked_fill(padded[:, None], 0.0))
