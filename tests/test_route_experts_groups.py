"""Groups that a wavefront's lanes do not hold are refused by the routing itself, with the reason, ahead of any launch."""
import pytest
import torch

from hibana_amd import _lib
from hibana_amd.kernels import ops


@pytest.mark.parametrize("groups,size,taken", [(33, 16, True), (33, 17, False), (63, 16, True), (60, 17, False), (17, 32, True), (17, 33, False), (31, 33, False), (9, 64, True), (9, 65, False),
                                               (5, 128, True), (5, 129, False), (3, 256, True), (3, 257, False), (64, 16, True), (2, 512, True), (1, 1024, True)])
def test_experts_of_a_group(groups, size, taken):
    logits = torch.zeros(2, groups * size)
    if groups * size > 1024:
        pytest.skip("more experts than any")
    with pytest.raises(RuntimeError if taken else ValueError, match="GPU only" if taken else f"{groups} groups"):
        ops.route_experts(logits, 1, groups=groups)  # (CPU tensors: what is not refused ends there)
    if not taken:
        e = groups * size
        assert _lib.lib().hb_route_experts(256, 2, e, 2, e, 1, 0, None, groups, 1, 1, 1.0, None, 1, 256, 256, None) == _lib.HB_EINVAL
