"""The ids that routed experts in the microscaled four-bit format take: whole numbers of any width, one outside the object's range adding nothing."""
import pytest
import torch

from oracle import mxfp4_format as om


def _experts(e, hidden, inter, device, base=0):
    from hibana_amd.kernels import mxfp4_moe
    g = torch.Generator().manual_seed(e)
    fc1, fc2 = (om.quantize(torch.randn(e, n, k, generator=g) / k ** 0.5) for n, k in ((2 * inter, hidden), (hidden, inter)))
    return mxfp4_moe.Mxfp4Experts(*(t.to(device) for t in (*fc1, *fc2)), base=base), fc1, fc2


def test_ids_that_are_no_whole_numbers_are_refused():
    from hibana_amd.kernels import mxfp4_moe
    ex, _, _ = _experts(4, 64, 32, "cpu")
    ex.tiled1 = ex.tiled2 = torch.zeros(1, dtype=torch.uint8)  # (not read: every call below is refused)
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 3)
    for kind in (torch.float32, torch.bfloat16, torch.bool, torch.complex64):
        with pytest.raises(ValueError):
            mxfp4_moe.mxfp4_moe(ex, x, torch.zeros(2, 3, dtype=kind), w)


def test_wide_ids_keep_outside():
    from hibana_amd.kernels.mxfp4_moe import _ids32
    wide = torch.tensor([[0, 3, 2**31 - 1], [2**31, 2**32 + 3, 2**40], [-1, -2**31 - 1, -2**33 + 2]])
    got = _ids32(wide.t())
    assert got.dtype == torch.int32 and got.is_contiguous()
    assert got.t().tolist() == [[0, 3, 2**31 - 1], [2**31 - 1] * 3, [-1] * 3]
    assert _ids32(torch.tensor([[1, 200]], dtype=torch.uint8)).tolist() == [[1, 200]]


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 40, 300])
def test_every_width_of_an_id(m):
    from hibana_amd.kernels import mxfp4_moe
    ex, fc1, fc2 = _experts(7, 128, 64, "cuda", base=3)
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, 128, generator=g).bfloat16(), torch.rand(m, 4, generator=g)
    ids = torch.randint(0, 14, (m, 4), generator=g)
    want = mxfp4_moe.mxfp4_moe(ex, x.cuda(), ids.int().cuda(), w.cuda())
    _, off = om.moe(x, ids, w, fc1, fc2, base=3)
    far = (want.double().cpu() - om.moe(x, ids, w, fc1, fc2, base=3)[0]).abs()
    assert bool((far <= off * 1.001 + 2.0 ** -8 * 1.01 * (want.double().cpu().abs() + off) * (1 + 2.0 ** -7) + 1e-30).all())
    for kind in (torch.int64, torch.int16, torch.int8, torch.uint8):
        assert torch.equal(want, mxfp4_moe.mxfp4_moe(ex, x.cuda(), ids.to(kind).cuda(), w.cuda()))
    inside = (ids >= 3) & (ids < 10)
    for shift in (2**32, -2**32, 2**40, 2**31):
        wide = torch.where(inside, ids, ids + shift)  # those outside stay outside ...
        assert torch.equal(want, mxfp4_moe.mxfp4_moe(ex, x.cuda(), wide.cuda(), w.cuda()))
        assert not mxfp4_moe.mxfp4_moe(ex, x.cuda(), (ids + shift).cuda(), w.cuda()).any()  # ... and so is every id so far off
