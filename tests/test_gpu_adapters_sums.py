"""The sums between an adapter's two products keep every bit that FP32 holds, in every type: differences of neighbouring 24-bit sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# x a^T = 2^23 + 4095 and 2^23 + 4094 (every partial sum a whole number below 2^24: exact in any order). In two parts of the type both are 2^23 + 4096, in FP32
# they are one apart, and so are their products with ones.
LEFT = [2048.0, 63.0, 1.0]
RIGHT = [[4096.0, 65.0, 0.0], [4096.0, 65.0, -1.0]]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [1, 40, 256, 300])
def test_result_and_rows_gradient(m, kind):
    from hibana_amd.kernels import adapters
    rows, matrix = torch.tensor(LEFT).expand(m, 3).to(kind).cuda(), torch.tensor([RIGHT]).to(kind).cuda()
    ends = torch.tensor([[[1.0], [-1.0]]]).expand(1, 2, 33).contiguous().to(kind).cuda()
    index = torch.zeros(m, dtype=torch.int32, device="cuda")
    out = adapters.add(torch.zeros(m, 33, dtype=kind, device="cuda"), rows, adapters.Adapters(matrix, ends), index)
    assert (out == 1).all()
    dx, _, _ = adapters.grads(rows, torch.zeros(m, 33, dtype=kind, device="cuda"), adapters.Adapters(ends, matrix), index)
    assert (dx == 1).all()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [2, 300])
def test_matrices_gradients(m, kind):
    """Two rows whose sums are one apart, times 1 and -1; all other rows are zeros."""
    from hibana_amd.kernels import adapters
    left, ends = torch.zeros(m, 3), torch.zeros(m, 33)
    left[:2] = torch.tensor([[2048.0, 63.0, 0.0], [2048.0, 63.0, 1.0]])
    ends[0], ends[1] = 1.0, -1.0
    left, ends = left.to(kind).cuda(), ends.to(kind).cuda()
    row, other = torch.tensor([[RIGHT[1]]]).to(kind).cuda(), torch.zeros(1, 1, 33, dtype=kind, device="cuda")
    index = torch.zeros(m, dtype=torch.int32, device="cuda")
    _, da, _ = adapters.grads(left, ends, adapters.Adapters(other, row), index)
    _, _, db = adapters.grads(ends, left, adapters.Adapters(row, other), index)
    assert (da == 1).all() and (db == 1).all()
