"""silu(gate) * up rounded to the microscaled four-bit format where the gate is next to nothing and the up value brings the product back: the codes
of the product in 64 bits."""
import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu


def _check(gate, up, dtype=torch.float32):
    from hibana_amd.kernels import ops
    x = torch.cat((gate, up), -1).to(dtype)
    got = ops.silu_mul_quant_mxfp4(x.cuda())
    want = om.quantize(om.silu_mul(x))
    assert torch.equal(got.scales.cpu(), want[1])
    assert torch.equal(got.codes.cpu(), want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_subnormal_gates_under_large_ups(dtype):
    g = torch.Generator().manual_seed(5)
    step = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133  # the type's smallest
    small = (torch.randint(1, 1024 if dtype == torch.float32 else 128, (256, 32), generator=g).double() * step).float()
    sign = torch.randint(0, 2, (256, 32), generator=g).float() * 2 - 1
    up = torch.exp2(100.0 + torch.rand(256, 32, generator=g)) * (torch.randint(0, 2, (256, 32), generator=g).float() * 2 - 1)
    _check(small * sign, up, dtype)
    alone = torch.zeros(256, 32)  # one such gate among zeros: the group's only value
    alone[torch.arange(256), torch.randint(0, 32, (256,), generator=g)] = small[:, 0]
    _check(alone, up, dtype)
    mixed = torch.where(torch.rand(256, 32, generator=g) < 0.5, small * sign, torch.randn(256, 32, generator=g) * 2.0 ** -126)
    _check(mixed, up, dtype)


def test_gates_around_the_border_of_the_short_way():
    """FP32 gates from the smallest to 2^-90, each exponent, mantissas at random and at the powers of two."""
    g = torch.Generator().manual_seed(6)
    e = torch.arange(-149, -89, dtype=torch.float64)[:, None]
    gate = torch.ldexp(1.0 + torch.rand(60, 32, generator=g, dtype=torch.float64) * (torch.arange(32) % 4 > 0), e.int()).float()
    for shift in (0.0, 13.0, 27.0):
        up = torch.exp2(-e - shift).clamp(max=2.0 ** 127).float() * (1.0 + torch.rand(60, 32, generator=g))
        _check(gate, up.clamp(max=3e38))
        _check(-gate, up.clamp(max=3e38))


def test_zero_gates_and_their_signs():
    gate = torch.zeros(4, 32)
    gate[1], gate[2, ::2], gate[3, 5] = -0.0, -0.0, 2.0 ** -149
    _check(gate, torch.full((4, 32), 2.0 ** 120))
    _check(gate, torch.full((4, 32), -1.0))
