"""`out` of the adapters' add among y's rows: refused by the library, unless it is y itself or lies between the rows. What is not refused ends at the launch,
for want of a device: the addresses are nobody's, so these run where there is no GPU alone."""
import ctypes as C
import itertools

import pytest
import torch

from hibana_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nothing is behind: for a machine without a GPU")

BASE = 1 << 20
POOL = C.byref(_lib.HbAdapters(256, 256, None, None, 2, 4, 8, 6, 0))  # BF16 [2, 4, 8], [2, 4, 6]
N, SIZE = 6, 2


def _call(y, y_stride, out, out_stride, m):
    return _lib.lib().hb_adapters_add(POOL, 256, 8, y, y_stride, 256, 4, m, out, out_stride, 1024, 1 << 40, None)


def _meet(y, y_stride, out, out_stride, m):
    rows = {y + SIZE * (r * y_stride + c) for r in range(m) for c in range(N)}
    return any(out + SIZE * (r * out_stride + c) in rows for r in range(m) for c in range(N))


@pytest.mark.parametrize("m", [1, 2, 5, 7])
def test_every_place_near_y(m):
    for y_stride, out_stride in itertools.product((6, 7, 11, 12, 13, 24, 25), repeat=2):
        for off in range(-(m + 1) * 30, (m + 1) * 30 + 1):
            same = off == 0 and y_stride == out_stride
            want = _lib.HB_EINVAL if not same and _meet(BASE, y_stride, BASE + SIZE * off, out_stride, m) else _lib.HB_ELAUNCH
            assert _call(BASE, y_stride, BASE + SIZE * off, out_stride, m) == want, (y_stride, out_stride, off)


def test_many_rows():
    m, stride = 1 << 24, 1 << 20
    assert _call(BASE, stride, BASE, stride, m) == _lib.HB_ELAUNCH
    assert _call(BASE, stride, BASE + SIZE * N, stride, m) == _lib.HB_ELAUNCH                       # beside y's columns
    assert _call(BASE, stride, BASE + SIZE * (N - 1), stride, m) == _lib.HB_EINVAL
    assert _call(BASE, stride, BASE + SIZE * stride * (m - 1), stride, m) == _lib.HB_EINVAL            # its first row is y's last
    assert _call(BASE, stride, BASE + SIZE * (stride * (m - 1) + N), stride, m) == _lib.HB_ELAUNCH
    assert _call(BASE, stride, BASE + SIZE * stride * m, N, m) == _lib.HB_ELAUNCH

