"""Linears in the microscaled four-bit format on both sides of the sizes at which a call is made another way: one or two tiles of weight rows a workgroup, the
rounding inside the product's launch or ahead of it, the ring."""
import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, n, k", [
    (1, 8192, 96), (5, 8193, 96), (32, 8224, 1056), (30, 8224, 2080), (32, 9000, 2080),          # 256, 257 and more tiles: one, two; inside, ahead
    (32, 16384, 1088), (3, 16390, 96), (30, 16416, 1632), (32, 16416, 1568), (20, 24570, 1056),  # 512, 513 and more: two, one
    (7, 24580, 96), (32, 24580, 1600), (30, 24580, 2208),                                        # past 768: two
    (32, 32768, 1024), (2, 32770, 64), (32, 32770, 1600), (30, 32770, 1632), (9, 40970, 96),     # past 1024: one, and the ring
    (160, 4000, 96), (128, 4000, 832), (129, 4000, 832), (300, 2000, 256), (1000, 33, 64)])      # passes of 32 rows
def test_linear_across_the_borders(m, n, k):
    from hibana_amd.kernels import mxfp4, ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    g = torch.Generator().manual_seed(m * n + k)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(117, 123, (n, k // 32), generator=g, dtype=torch.uint8)
    x = (torch.randn(m, k, generator=g) * 0.125).bfloat16()
    lin = Mxfp4Linear(codes.cuda(), scales.cuda())
    got = ops.mxfp4_linear(x.cuda(), lin)
    x64, w64 = om.through(x), om.dequantize(codes, scales)
    want = x64 @ w64.T
    # sums of k exact products in FP32, in any order, and one rounding to BF16
    bound = k * 2.0 ** -24 * (x64.abs() @ w64.abs().T) + 2.0 ** -8 * 1.01 * want.abs()
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    held = ops.mxfp4_linear(mxfp4.quantize(x.cuda()), lin)
    off = (held.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    for _ in range(2):
        assert torch.equal(got, ops.mxfp4_linear(x.cuda(), lin))
