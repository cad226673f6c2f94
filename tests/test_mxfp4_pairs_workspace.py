"""The room that routed experts in the microscaled four-bit format take where the caller's own tensor holds the pairs' outputs."""
import ctypes as C

import pytest
import torch

from hibana_amd import _lib


def _experts(experts=16, hidden=256, inter=128, hidden_out=2048, gated=1):
    return _lib.HbMxfp4Experts(256, 256, experts, 0, hidden, inter, hidden_out, gated)


@pytest.mark.parametrize("m, k", [(1, 4), (9, 8), (100, 4), (1024, 8), (1 << 20, 8)])  # one launch a product, the plan's slots, the ring, passes
def test_pairs_need_no_room_for_a_sums(m, k):
    lib, ex = _lib.lib(), _experts()
    whole, pairs = lib.hb_mxfp4_moe_workspace_bytes(C.byref(ex), m, k), lib.hb_mxfp4_moe_pairs_workspace_bytes(C.byref(ex), m, k)
    assert 0 < pairs and whole - pairs == min(m * k, 1 << 18) * 2048 * 4
    call = lambda mode, size: lib.hb_mxfp4_moe(C.byref(ex), 256, 256, 256, m, k, mode, 256, 256, size, None)  # noqa: E731
    assert call(0, whole - 1) == call(1, pairs - 1) == call(2, pairs - 1) == _lib.HB_EWORKSPACE  # (before a launch)


def test_sizes_that_are_refused():
    lib, ex = _lib.lib(), _experts()
    for m, k in [(0, 2), (4, 0), (4, 4097), (1 << 30, 2)]:
        assert lib.hb_mxfp4_moe_pairs_workspace_bytes(C.byref(ex), m, k) == 0
    assert lib.hb_mxfp4_moe_pairs_workspace_bytes(None, 4, 2) == lib.hb_mxfp4_moe_pairs_workspace_bytes(C.byref(_experts(hidden=48)), 4, 2) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 300, 2048])
def test_a_call_for_pairs_allocates_them_once(m):
    from hibana_amd.kernels import mxfp4_moe
    g = torch.Generator(device="cuda").manual_seed(m)
    ex = mxfp4_moe.Mxfp4Experts.from_dense(*(torch.randn(*s, device="cuda", generator=g) / 16 for s in ((16, 256, 256), (16, 2048, 128))))
    mxfp4_moe.tile(ex, release=True)
    x = torch.randn(m, 256, device="cuda", generator=g).bfloat16()
    w, ids = torch.topk(torch.randn(m, 16, device="cuda", generator=g), 8)
    w, ids = torch.softmax(w, -1), ids.int()
    summed = mxfp4_moe.mxfp4_moe(ex, x, ids, w)  # beside it: the sizes of the two are kept apart
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    pairs = mxfp4_moe.mxfp4_moe(ex, x, ids, w, pairs=True)
    assert torch.cuda.max_memory_allocated() - before < 1.5 * pairs.numel() * 4 + (1 << 20)
    assert torch.equal(pairs, mxfp4_moe.mxfp4_moe(ex, x, ids, w, pairs=True))
    assert torch.equal(summed, mxfp4_moe.mxfp4_moe(ex, x, ids, w))
    half = mxfp4_moe.mxfp4_moe(ex, x, ids, w, pairs=True, pairs_bf16=True)
    assert torch.equal(half, pairs.bfloat16())
