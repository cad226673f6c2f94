"""Calls that find microscaled four-bit weights not laid out yet, on streams that know nothing of each other."""
import threading

import pytest
import torch

from oracle import mxfp4_format as om

pytestmark = pytest.mark.gpu


def _held(n, k, seed, stack=()):
    g = torch.Generator().manual_seed(seed)
    return tuple(t.cuda() for t in om.quantize(torch.randn(*stack, n, k, generator=g) / k ** 0.5))


def _busy():
    """Some milliseconds of work on the current stream."""
    x = torch.zeros(1 << 28, device="cuda")
    for _ in range(20):
        x.add_(1.0)


def _linear():
    from hibana_amd.kernels import ops
    from hibana_amd.weights.mxfp4 import Mxfp4Linear
    x = torch.randn(9, 1024, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    lin = Mxfp4Linear(*_held(3000, 1024, 2))
    return lin, lambda: ops.mxfp4_linear(x, lin)


def _experts():
    from hibana_amd.kernels import mxfp4_moe
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 512, generator=g).bfloat16().cuda()
    w, ids = (t.cuda() for t in torch.topk(torch.randn(20, 24, generator=g), 4))
    ex = mxfp4_moe.Mxfp4Experts(*_held(512, 512, 4, (24,)), *_held(512, 256, 5, (24,)))
    return ex, lambda: mxfp4_moe.mxfp4_moe(ex, x, ids, torch.softmax(w, -1))


@pytest.mark.parametrize("make", [_linear, _experts])
def test_the_second_call_on_another_stream(make):
    _, call = make()
    want = call()
    _, call = make()  # the same weights, not laid out
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _busy()
        first = call()
    second = call()  # on a stream that waits for nothing
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("make", [_linear, _experts])
def test_first_calls_of_two_threads(make):
    _, call = make()
    want = call()
    _, call = make()
    torch.cuda.synchronize()
    got, start = [None, None], threading.Barrier(2)

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            got[i] = [call() for _ in range(3)]

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for ys in got for y in ys)


def test_released_rows_may_be_overwritten_at_once():
    """`release` on a side stream: the memory of the codes goes back to the stream that they came from, which uses it again."""
    lin, call = _linear()
    want = call()
    lin, call = _linear()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _busy()
        lin.tile(release=True)
    taken = [torch.full((3000 * 512,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
    got = call()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(bool((t == 255).all()) for t in taken)
