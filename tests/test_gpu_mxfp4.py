"""The microscaled four-bit operators on the GPU against the FP64 oracle: the rounding and its values bit for bit, the product to the
error of an FP32 sum and one rounding."""
import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # of a rounding, relative


def _same(q, want):
    assert torch.equal(q.scales.cpu(), want[1])
    assert torch.equal(q.codes.cpu(), want[0])


def _values(rows, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, max(1, k // 32)), generator=g).float()).repeat_interleave(32, -1)
    x.view(-1)[:: 37] = 0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, k", [(1, 32), (1, 96), (3, 5120), (77, 4128), (1543, 160)])
def test_rounding_is_the_definitions(rows, k, dtype):
    from hibana_amd.kernels import mxfp4
    x = _values(rows, k, dtype, rows * k)
    q = mxfp4.quantize(x.cuda())
    want = om.quantize(x)
    _same(q, want)
    for to in TYPES:
        assert torch.equal(mxfp4.dequantize(q, to).cpu(), om.dequantize(*want).to(to))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value_of_a_sixteen_bit_type(dtype):
    """Each bit pattern among a group's others under several largest magnitudes; a group with a non-finite value is NaN whole."""
    from hibana_amd.kernels import mxfp4
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    alone = every[:, None].expand(-1, 32).contiguous()  # its own scale
    _same(mxfp4.quantize(alone.cuda()), om.quantize(alone))
    for top in (1.0, 5.5, 7.0, 96.0, 2.0 ** -14):
        x = every.view(-1, 16).repeat(1, 2)
        x[:, 16:] = top
        _same(mxfp4.quantize(x.cuda()), om.quantize(x))


def test_borders_subnormals_and_extremes_in_fp32():
    from hibana_amd.kernels import mxfp4
    x = torch.zeros(254 + 24, 32)
    for e in range(-150, 128):  # a group whose largest has exponent e: borders between codes and the values next to them
        unit = 2.0 ** (e - 2)
        border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 4.0], dtype=torch.float64) * unit
        at = border.float()
        row = torch.cat((at, torch.nextafter(at, torch.tensor(0.0)), -torch.nextafter(at, torch.tensor(float("inf"))), torch.tensor([0.0, -0.0])))
        x[e + 150] = torch.where(torch.isfinite(row), row, torch.zeros(()))
    _same(mxfp4.quantize(x.cuda()), om.quantize(x))
    assert torch.equal(mxfp4.dequantize(mxfp4.quantize(x.cuda())).cpu().double(), om.through(x))


def test_groups_that_are_not_finite_stand_for_nan():
    from hibana_amd.kernels import mxfp4
    x = torch.ones(4, 128)
    x[0, 5], x[1, 40], x[2, 127], x[3] = float("inf"), float("nan"), float("-inf"), float("nan")
    q = mxfp4.quantize(x.cuda())
    _same(q, om.quantize(x))
    back = mxfp4.dequantize(q, torch.bfloat16).cpu()
    assert torch.equal(back.isnan(), om.through(x).isnan()) and int(back.isnan().sum()) == 3 * 32 + 128


def test_dequantize_takes_every_code_and_scale():
    from hibana_amd.kernels import mxfp4
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    codes = (torch.arange(16, dtype=torch.uint8) | torch.arange(15, -1, -1, dtype=torch.uint8) << 4).expand(256, 16).contiguous()
    want = om.dequantize(codes, scales)
    for to in TYPES:
        got = mxfp4.dequantize(mxfp4.Mxfp4(codes.cuda(), scales.cuda()), to).cpu()
        expected = want.float().to(to)  # (a value past FP32's range is an infinity there)
        assert torch.equal(got.isnan(), expected.isnan()) and torch.equal(got.nan_to_num(0.0), expected.nan_to_num(0.0))


def test_leading_axes_strides_offsets_and_nothing():
    from hibana_amd.kernels import mxfp4
    x = _values(24, 256, torch.bfloat16, 5)
    q = mxfp4.quantize(x.cuda().view(2, 3, 4, 256))
    assert q.codes.shape == (2, 3, 4, 128) and q.scales.shape == (2, 3, 4, 8) and q.shape == (2, 3, 4, 256)
    _same(mxfp4.Mxfp4(q.codes.flatten(0, 2), q.scales.flatten(0, 2)), om.quantize(x))
    wide = _values(24, 320, torch.bfloat16, 6).cuda()
    _same(mxfp4.quantize(wide[:, 32:288]), om.quantize(wide[:, 32:288].cpu()))
    _same(mxfp4.quantize(wide[::2]), om.quantize(wide[::2].cpu()))
    odd = torch.zeros(24 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(24, 256)  # starts off the 16-byte boundary
    odd.copy_(x)
    _same(mxfp4.quantize(odd), om.quantize(x))
    part = mxfp4.Mxfp4(q.codes.flatten(0, 2)[::3, 16:64], q.scales.flatten(0, 2)[::3, 1:4])
    assert torch.equal(mxfp4.dequantize(part).cpu().double(), om.dequantize(part.codes.cpu(), part.scales.cpu()))
    import copy
    import pickle
    for other in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), mxfp4.Mxfp4(*q)):
        assert other.shape == q.shape and torch.equal(mxfp4.dequantize(other), mxfp4.dequantize(q))
    for shape in ((0, 64), (5, 0), (0,)):
        e = mxfp4.quantize(torch.empty(shape, device="cuda"))
        assert mxfp4.dequantize(e).shape == shape


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, half, pairs", [(1, 32, 0), (4, 25600, 0), (5, 96, 32), (33, 512, 64), (7, 160, 8), (300, 4128, 0)])
def test_gated_product_rounds_as_the_exact_one(rows, half, pairs, dtype):
    from hibana_amd.kernels import ops
    x = _values(rows, 2 * half, dtype, half + rows) * 0.25
    _same(ops.silu_mul_quant_mxfp4(x.cuda(), pairs), om.quantize(om.silu_mul(x, pairs)))


def test_gated_product_at_the_ends_of_the_range():
    """Gates whose exponential leaves FP32, products that are subnormal or nothing, products that land on a border or on the
    power of two that sets the scale, products past FP32, non-finite factors."""
    from hibana_amd.kernels import ops
    g = torch.Generator().manual_seed(3)
    gate = torch.randn(40, 32, generator=g)
    up = torch.randn(40, 32, generator=g)
    gate[0], gate[1], gate[2], gate[3] = -100.0, -89.5, 3e38, -3e38
    up[2] = 1e-38 * torch.randn(32, generator=g)
    gate[4], up[4] = 1e-30, 1e-30
    gate[5], up[5] = 1e-25, 1e-14
    gate[6] = 1e-20 * torch.rand(32, generator=g)  # silu(g) = g / 2
    up[6] = 1e-18
    gate[7], up[7] = 200.0, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4) / 200.0  # silu(200) is 200 in FP32, a little less in truth
    gate[8], up[8] = 3e30, 3e30
    gate[9, 3], gate[10, 3], gate[11, 3], up[12, 3], up[13, 3] = float("inf"), float("-inf"), float("nan"), float("inf"), float("nan")
    gate[14], up[14] = 0.0, -1.0
    gate[15, 1:] = 0.0
    gate[16:], up[16:] = 64.0 + torch.rand(24, 32, generator=g), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4) / 64
    x = torch.cat((gate, up), -1)
    _same(ops.silu_mul_quant_mxfp4(x.cuda()), om.quantize(om.silu_mul(x)))


def test_gated_product_of_a_million_values():
    """Enough values for some to lie within FP32's error of a border: every code is the exact product's."""
    from hibana_amd.kernels import ops
    g = torch.Generator().manual_seed(9)
    x = torch.randn(512, 2 * 8192, generator=g) * 2
    _same(ops.silu_mul_quant_mxfp4(x.cuda()), om.quantize(om.silu_mul(x)))


def _weight(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(117, 123, (n, k // 32), generator=g, dtype=torch.uint8)
    return codes, scales


def _check_product(got, x64, w64, dtype):
    """Sums of k products in FP32 (each exact, k additions at most, in any order) and one rounding: off by at most
    k 2^-24 sum |x w| and half a step of the result."""
    want = x64 @ w64.T
    bound = x64.shape[1] * 2.0 ** -24 * (x64.abs() @ w64.abs().T) + HALF_STEP[dtype] * want.abs() * 1.01 + 2.0 ** -25 * (dtype == torch.float16)
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(1, 1, 32), (1, 5120, 5120), (2, 17, 96), (5, 33, 128), (8, 640, 2688), (15, 1000, 544), (16, 64, 4096), (17, 80, 160),
                                     (31, 257, 1056), (64, 512, 512), (77, 1024, 2080), (128, 129, 640), (200, 96, 1024), (300, 777, 288), (20, 24600, 2560),
                                     (2048, 5120, 96), (16, 64, 8192), (130, 130, 4128), (40, 33, 5152), (3, 16416, 96), (7, 16411, 2080), (2048, 8500, 96), (1025, 16500, 64),
                                     (32, 77, 16384), (30, 24610, 3008), (64, 3000, 4160), (90, 2001, 4128), (128, 2050, 4160), (1100, 9001, 544)])
def test_linear(m, n, k, dtype):
    from hibana_amd.kernels import mxfp4, ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    codes, scales = _weight(n, k, n + k)
    x = _values(m, k, dtype, m + k) * 0.125
    lin = Mxfp4Linear(codes.cuda(), scales.cuda())
    got = ops.mxfp4_linear(x.cuda(), lin)
    assert got.dtype == dtype and got.shape == (m, n)
    x64, w64 = om.through(x), om.dequantize(codes, scales)
    _check_product(got, x64, w64, dtype)
    held = ops.mxfp4_linear(mxfp4.quantize(x.cuda()), lin, dtype)  # rounded beforehand: the same operands
    _check_product(held, x64, w64, dtype)
    assert torch.equal(got, ops.mxfp4_linear(x.cuda(), lin))  # repeatable


def test_weights_layout_and_the_way_back():
    from hibana_amd.kernels import mxfp4
    from hibana_amd.weights.linear import Linear
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    for n, k in [(1, 32), (16, 128), (33, 544), (640, 5120)]:
        codes, scales = _weight(n, k, n)
        lin = Mxfp4Linear(codes.cuda(), scales.cuda()).tile(release=True)
        assert isinstance(lin, Linear) and lin.codes is None and (lin.out_features, lin.in_features) == (n, k) and lin.bytes == n * k // 2 + n * k // 32
        assert torch.equal(lin.held.codes.cpu(), codes) and torch.equal(lin.held.scales.cpu(), scales)
        assert torch.equal(lin.dequantize().cpu().double(), om.dequantize(codes, scales))
    for inter, k in [(32, 64), (160, 288)]:
        stack = [_weight(2 * inter, k, s) for s in range(3)]
        q = mxfp4.Mxfp4(torch.stack([c for c, _ in stack]).cuda(), torch.stack([s for _, s in stack]).cuda())
        back = mxfp4.untile(mxfp4.tile(q, gated=True), 2 * inter, k, gated=True)
        assert torch.equal(back.codes, q.codes) and torch.equal(back.scales, q.scales)
    w = _values(48, 96, torch.bfloat16, 1)
    assert torch.equal(Mxfp4Linear.from_dense(w.cuda()).dequantize().cpu().double(), om.through(w))


def test_a_row_that_is_not_finite_stays_among_itself():
    from hibana_amd.kernels import ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    codes, scales = _weight(48, 256, 4)
    lin = Mxfp4Linear(codes.cuda(), scales.cuda())
    for m in (3, 16, 40):
        x = _values(m, 256, torch.bfloat16, m) * 0.125
        x[1, 70] = float("inf")
        got = ops.mxfp4_linear(x.cuda(), lin)
        assert bool(got[1].isnan().all())
        keep = [i for i in range(m) if i != 1]
        _check_product(got[keep], om.through(x[keep]), om.dequantize(codes, scales), torch.bfloat16)


def test_other_streams_and_a_captured_graph():
    from hibana_amd.kernels import mxfp4, ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    up = Mxfp4Linear(*(t.cuda() for t in _weight(512, 256, 1))).tile()
    down = Mxfp4Linear(*(t.cuda() for t in _weight(256, 256, 2))).tile()

    def block(x):  # the operators in a row, as a dense block uses them
        return ops.mxfp4_linear(ops.silu_mul_quant_mxfp4(ops.mxfp4_linear(x, up)), down), mxfp4.dequantize(mxfp4.quantize(x))

    for m in (1, 9, 70):
        x = _values(m, 256, torch.bfloat16, m).cuda() * 0.03
        eager = block(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = block(x)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(eager, there))
        held = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(held)
        for seed in range(3):
            fresh = _values(m, 256, torch.bfloat16, 100 + seed).cuda() * 0.03
            held.copy_(fresh)
            graph.replay()
            want = block(fresh)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
