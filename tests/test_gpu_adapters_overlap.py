"""`out` of `adapters.add`: y itself, columns or rows between y's, memory of x; anything that shares a part of y's rows is refused and left as it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [5, 300])
def test_out_beside_and_among_the_rows(m):
    from hibana_amd.kernels import adapters
    g = torch.Generator().manual_seed(m)
    pool = adapters.Adapters(torch.randn(2, 4, 24, generator=g).cuda(), torch.randn(2, 4, 24, generator=g).cuda())
    buffer, x, index = torch.randn(2 * m + 2, 80, generator=g).cuda(), torch.randn(m, 24, generator=g).cuda(), (torch.arange(m) % 3 - 1).cuda()
    y = buffer[:m, 5:29]
    want, before = adapters.add(y, x, pool, index), buffer.clone()
    for out in (buffer[:m, 6:30], buffer[:m, 4:28], buffer[:m, 28:52], buffer[1:m + 1, 5:29], buffer[m - 1:2 * m - 1, 28:52], buffer.view(-1)[10:10 + 81 * m].view(m, 81)[:, :24],
                buffer.view(-1)[5:5 + 24 * m].view(m, 24)):
        with pytest.raises(ValueError):
            adapters.add(y, x, pool, index, out=out)
        assert torch.equal(buffer, before)
    for out in (buffer[:m, 29:53], buffer[1:m + 1, 29:53], buffer[m:2 * m, 5:29], buffer[:2 * m:2, 40:64], y):
        buffer.copy_(before)
        assert torch.equal(adapters.add(y, x, pool, index, out=out), want)
        left = before.clone()
        left.as_strided(out.shape, out.stride(), out.storage_offset()).copy_(want)
        assert torch.equal(buffer, left)
    assert torch.equal(adapters.add(before[:m, 5:29], x, pool, index, out=x), want)  # x is read before out is written
