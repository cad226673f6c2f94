"""The dense MLP on three-bit copies with adapters beside it: a request without one has the base model's bits, whatever else is in the batch."""
import pytest
import torch

from tests.test_gpu_adapted_layers import _mxfp4, _nvfp4, _pool

pytestmark = pytest.mark.gpu


@pytest.fixture
def three_bit():
    from hibana_amd.kernels import w3
    w3.set_enabled(True)
    yield
    w3.set_enabled(None)


def _linears(form, pairs):
    from hibana_amd.kernels import w3
    lins = (_mxfp4(512, 128, 4, pairs), _mxfp4(128, 256, 5)) if form == "mxfp4" else (_nvfp4(512, 128, 4), _nvfp4(128, 256, 5))
    if form != "mxfp4":
        lins[0].pairs = pairs
        w3.attach([(str(i), lin) for i, lin in enumerate(lins) if form == "w3" or form == "w3 down" and i], "lloyd")
    return lins


@pytest.mark.parametrize("m", [1, 9, 40, 128, 129])
@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("pairs", [0, 32])
@pytest.mark.parametrize("form", ["w3", "w3 down", "nvfp4", "mxfp4"])
def test_requests_without_an_adapter(form, pairs, which, m, three_bit):
    from hibana_amd.model.mlp import Mlp
    lins = _linears(form, pairs)
    mlp = Mlp(*lins, adapters=tuple(_pool(lin.in_features, lin.out_features, 6 + i) if on else None for i, (lin, on) in enumerate(zip(lins, which))))
    x = torch.randn(m, 128, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    base, index = mlp(x), (torch.arange(m) % 4 - 1).cuda()
    assert torch.equal(mlp(x, index=torch.full((m,), -1, device="cuda")), base)
    got = mlp(x, index=index)
    assert torch.equal(got[index < 0], base[index < 0]) and (m == 1 or torch.equal(got, base) == (not any(which)))


@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("pairs", [0, 32])
def test_rows_with_adapters(pairs, which, m, three_bit):
    """The down projection's base reads the rounded groups, as without adapters; its adapters the product ahead of that rounding."""
    from hibana_amd.kernels import adapters, ops, w3
    from hibana_amd.model.mlp import Mlp
    lins = _linears("w3", pairs)
    pools = tuple(_pool(lin.in_features, lin.out_features, 6 + i) if on else None for i, (lin, on) in enumerate(zip(lins, which)))
    x = torch.randn(m, 128, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    index = (torch.arange(m) % 4 - 1).cuda()
    gate_up = w3.w3_linear(x, lins[0].w3)
    gate_up = gate_up if pools[0] is None else adapters.add(gate_up, x, pools[0], index)
    codes, scales = ops.silu_mul_quant_groups(gate_up, pairs, torch_chain=True)
    y = w3.w3_linear(codes, lins[1].w3, scales)
    want = y if pools[1] is None else adapters.add(y, ops.silu_and_mul(gate_up, pairs), pools[1], index)
    assert torch.equal(Mlp(*lins, adapters=pools)(x, index=index), want)
