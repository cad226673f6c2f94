"""The microscaled four-bit operators where offsets and counts pass 32 bits: rows far behind the first, weights past 4 GiB, launches and
passes that have to be split. Rows at the ends and at the borders against the FP64 oracle; memory is the only size that matters here."""
import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu


def _need(gib):
    free = torch.cuda.mem_get_info()[0] >> 30
    if free < gib + 4:
        pytest.skip(f"{free} GiB of device memory free, {gib} needed")


def _near(got, want, off, half_step=2.0 ** -8):
    far = (got.double().cpu() - want).abs()
    bound = off * 1.001 + half_step * 1.01 * (want.abs() + off) + 1e-30
    assert bool((far <= bound).all()), float((far / bound).max())


def _fill(x, rows, seed):
    """Random values in the named rows of a zero tensor on the GPU -> those rows on the CPU."""
    g = torch.Generator().manual_seed(seed)
    some = torch.randn(len(rows), x.shape[1], generator=g).to(x.dtype)
    x[torch.tensor(rows, device=x.device)] = some.cuda()
    return some


def test_rounding_of_more_lanes_than_a_launch_holds():
    """2^35 values and a row: a launch of eight values a lane would have 2^32 lanes and more."""
    from hibana_amd.kernels import mxfp4, ops
    k, rows = 1 << 18, (1 << 17) + 1
    _need(64 + 18)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    at = [0, 1 << 16, (1 << 16) - 1, rows - 2, rows - 1]
    some = _fill(x, at, 1)
    q = mxfp4.quantize(x)
    want = om.quantize(some)
    assert torch.equal(q.codes[at].cpu(), want[0]) and torch.equal(q.scales[at].cpu(), want[1])
    assert not q.codes[1: 1 << 15].any() and not q.scales[rows // 2 + 5: rows - 3].any()
    back = mxfp4.dequantize(q, torch.bfloat16)
    assert torch.equal(back[at].cpu().double(), om.dequantize(*want))
    del q, back
    h = ops.silu_mul_quant_mxfp4(x, 0)
    want = om.quantize(om.silu_mul(some))
    assert torch.equal(h.codes[at].cpu(), want[0]) and torch.equal(h.scales[at].cpu(), want[1])


@pytest.mark.parametrize("m, n, k, gib", [((1 << 20) + 7, 32, 4128, 14), ((1 << 18) + 5, 8200, 64, 6)])
def test_rows_and_results_past_32_bits(m, n, k, gib):
    from hibana_amd.kernels import ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    _need(gib)
    assert m * max(n, k) > 1 << 31
    w = om.quantize(torch.randn(n, k, generator=torch.Generator().manual_seed(2)) / k ** 0.5)
    lin = Mxfp4Linear(*(t.cuda() for t in w)).tile()
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    at = [0, 31, (1 << 32) // k if (1 << 32) // k < m else m // 2, (1 << 31) // n if (1 << 31) // n < m else m // 3, m - 33, m - 2, m - 1]
    some = _fill(x, at, 3)
    y = ops.mxfp4_linear(x, lin)
    x64, w64 = om.through(some), om.dequantize(*w)
    _near(y[at], x64 @ w64.T, k * 2.0 ** -24 * (x64.abs() @ w64.abs().T))
    named = torch.zeros(m, dtype=torch.bool, device="cuda")
    named[at] = True
    assert not y[~named].any()


@pytest.mark.parametrize("m", [1, 20, 150])
def test_weights_past_four_gib(m):
    from hibana_amd.kernels import ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    n, k = (1 << 19) + 40, 1 << 14
    _need(14)
    g = torch.Generator(device="cuda").manual_seed(4)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    scales = torch.randint(110, 121, (n, k // 32), generator=g, dtype=torch.uint8, device="cuda")
    at = [0, 100, n // 2, n - 41, n - 40, n - 1]
    w64 = om.dequantize(codes[at].cpu(), scales[at].cpu())
    lin = Mxfp4Linear(codes, scales).tile(release=True)
    del codes, scales
    assert lin.tiled.numel() > 1 << 32
    held = lin.held
    assert torch.equal(om.dequantize(held.codes[at].cpu(), held.scales[at].cpu()), w64)
    del held
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).bfloat16()
    y = ops.mxfp4_linear(x.cuda(), lin)
    x64 = om.through(x)
    _near(y[:, at], x64 @ w64.T, k * 2.0 ** -24 * (x64.abs() @ w64.abs().T))


@pytest.mark.parametrize("m", [2, 33, 200])
def test_experts_past_four_gib(m):
    from hibana_amd.kernels import mxfp4_moe
    e, hidden, inter = 250, 4096, 8192
    _need(40)
    g = torch.Generator(device="cuda").manual_seed(5)
    make = lambda *s: (torch.randint(0, 256, (*s[:-1], s[-1] // 2), generator=g, dtype=torch.uint8, device="cuda"),  # noqa: E731
                       torch.randint(112, 117, (*s[:-1], s[-1] // 32), generator=g, dtype=torch.uint8, device="cuda"))
    fc1, fc2 = make(e, 2 * inter, hidden), make(e, hidden, inter)
    named = [0, 61, 249]
    few = [tuple(t[named].cpu() for t in fc) for fc in (fc1, fc2)]
    ex = mxfp4_moe.tile(mxfp4_moe.Mxfp4Experts(*fc1, *fc2), release=True)
    del fc1, fc2
    assert ex.tiled1.numel() > 1 << 32 and ex.tiled2.numel() > 1 << 32
    h = torch.Generator().manual_seed(m)
    x = (torch.randn(m, hidden, generator=h) / 16).bfloat16()
    which = torch.randint(0, 3, (m, 2), generator=h)
    w = torch.softmax(torch.randn(m, 2, generator=h), -1)
    got = mxfp4_moe.mxfp4_moe(ex, x.cuda(), torch.tensor(named)[which].to(torch.int32).cuda(), w.cuda())
    _near(got, *om.moe(x, which, w, *few))


@pytest.mark.parametrize("gated", [True, False])
def test_a_call_of_several_passes(gated):
    """More pairs than a pass takes: each row's result is that of a call of its own part, whichever pass it fell into."""
    from hibana_amd.kernels import mxfp4_moe
    e, hidden, inter, k, m = 6, 32, 32, 4, (1 << 19) * 2 + 1300
    fc1 = om.quantize(torch.randn(e, 2 * inter if gated else inter, hidden, generator=torch.Generator().manual_seed(6)) / 6)
    fc2 = om.quantize(torch.randn(e, hidden, inter, generator=torch.Generator().manual_seed(7)) / 6)
    ex = mxfp4_moe.Mxfp4Experts(*(t.cuda() for t in (*fc1, *fc2)))
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(m, hidden, generator=g, device="cuda").bfloat16()
    ids = torch.randint(-1, e + 1, (m, k), generator=g, dtype=torch.int32, device="cuda")
    w = torch.rand(m, k, generator=g, device="cuda")
    got = mxfp4_moe.mxfp4_moe(ex, x, ids, w)
    pairs = mxfp4_moe.mxfp4_moe(ex, x, ids, w, pairs=True)
    named = ((ids >= 0) & (ids < e)).flatten()
    for lo in (0, (1 << 19) - 700, (1 << 20) - 650, m - 1300):
        part = slice(lo, lo + 1300)
        assert torch.equal(got[part], mxfp4_moe.mxfp4_moe(ex, x[part], ids[part], w[part]))
        of = slice(lo * k, (lo + 1300) * k)
        assert torch.equal(pairs[of][named[of]], mxfp4_moe.mxfp4_moe(ex, x[part], ids[part], w[part], pairs=True)[named[of]])
    at = slice(m - 40, m)
    y, off = om.moe_pairs(x[at].cpu(), ids[at].cpu(), fc1, fc2)
    want, far = om.moe(x[at].cpu(), ids[at].cpu(), w[at].cpu(), fc1, fc2)
    _near(got[at], want, far + 2.0 ** -8 * ((y.abs() + off) * w[at].cpu().double()[..., None]).sum(1))  # (pairs in BF16)
