"""What the microscaled four-bit operators refuse, on the CPU: nothing is launched."""
import ctypes as C

import pytest
import torch

from hibana_amd import _lib
from hibana_amd.kernels import mxfp4, ops
from hibana_amd.weights.mxfp4 import Mxfp4Linear


def test_the_library_refuses_before_a_launch():
    lib = _lib.lib()
    assert lib.hb_mxfp4_quantize(None, 0, 1, 32, 256, 256, None) == _lib.HB_ENULL
    for kind, rows, k, x, codes in [(3, 1, 32, 256, 256), (-1, 1, 32, 256, 256), (0, 0, 32, 256, 256), (0, 1, 48, 256, 256), (0, 1, 0, 256, 256), (0, 1, 32, 258, 256),
                                    (0, 1, 32, 256, 264), (0, 1 << 41, 32, 256, 256), (0, -1, 32, 256, 256)]:
        assert lib.hb_mxfp4_quantize(x, kind, rows, k, codes, 256, None) == _lib.HB_EINVAL
        assert lib.hb_mxfp4_dequantize(codes, 256, rows, k, kind, x, None) == _lib.HB_EINVAL
    assert lib.hb_mxfp4_dequantize(256, None, 1, 32, 0, 256, None) == _lib.HB_ENULL
    assert lib.hb_silu_mul_quant_mxfp4(256, 0, 1, 64, 0, None, 256, None) == _lib.HB_ENULL
    for half, pairs in [(48, 0), (64, 12), (64, -8), (96, 64), (0, 0)]:
        assert lib.hb_silu_mul_quant_mxfp4(256, 0, 1, half, pairs, 256, 256, None) == _lib.HB_EINVAL
    assert lib.hb_mxfp4_tiled_bytes(32, 64) == 1024 + 512 and lib.hb_mxfp4_tiled_bytes(33, 544) == 2 * 9 * 1024 + 2 * 4 * 256
    assert lib.hb_mxfp4_tiled_bytes(0, 128) == 0 and lib.hb_mxfp4_tiled_bytes(16, 48) == 0 and lib.hb_mxfp4_tiled_bytes(1 << 31, 32) == 0
    assert lib.hb_mxfp4_repack(256, 256, 1, 96, 128, 1, 256, None) == _lib.HB_EINVAL  # gated rows go in units of 64
    assert lib.hb_mxfp4_repack(256, 256, 65536, 64, 128, 0, 256, None) == _lib.HB_EINVAL
    assert lib.hb_mxfp4_unpack(None, 1, 64, 128, 0, 256, 256, None) == _lib.HB_ENULL
    need = lib.hb_mxfp4_linear_workspace_bytes(4, 64, 128, 0)
    call = lambda **c: lib.hb_mxfp4_linear(*{**dict(x=256, xs=None, kind=0, m=4, w=256, n=64, k=128, y=256, to=0, ws=256, size=max(need, 1 << 20), stream=None), **c}.values())  # noqa: E731
    assert call(x=None) == call(w=None) == call(y=None) == call(kind=3) == _lib.HB_ENULL
    for c in [dict(m=0), dict(m=(1 << 24) + 1), dict(n=0), dict(k=33), dict(kind=1), dict(kind=4), dict(to=3), dict(x=264), dict(w=257), dict(y=257)]:
        assert call(**c) == _lib.HB_EINVAL, c


def test_python_refusals():
    bf = torch.zeros(2, 64, dtype=torch.bfloat16)
    for bad in (torch.zeros(2, 64, dtype=torch.int32), torch.zeros(2, 64, dtype=torch.float64), torch.zeros(2, 48), torch.zeros(())):
        with pytest.raises(ValueError):
            mxfp4.quantize(bad)
    with pytest.raises(RuntimeError):
        mxfp4.quantize(bf)  # no CPU path
    held = mxfp4.Mxfp4(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        mxfp4.dequantize(held)
    with pytest.raises(ValueError):
        mxfp4.dequantize(held, torch.float64)
    for codes, scales in [(held.codes, held.scales[:, :1]), (held.codes.int(), held.scales), (held.codes[:, :8], held.scales[:, :1]), (held.codes, held.scales.int())]:
        with pytest.raises(ValueError):
            mxfp4.dequantize(mxfp4.Mxfp4(codes, scales))
        with pytest.raises(ValueError):
            Mxfp4Linear(codes, scales)
    with pytest.raises(ValueError):
        Mxfp4Linear(torch.zeros(2, 3, 32, dtype=torch.uint8), torch.zeros(2, 3, 2, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        Mxfp4Linear(*held).tile()
    for bad, pairs in [(torch.zeros(2, 96), 0), (torch.zeros(2, 128, dtype=torch.float64), 0), (torch.zeros(2, 128), 12), (torch.zeros(2, 192), 64), (torch.zeros(2, 128), -8)]:
        with pytest.raises(ValueError):
            ops.silu_mul_quant_mxfp4(bad, pairs)
    with pytest.raises(RuntimeError):
        ops.silu_mul_quant_mxfp4(torch.zeros(2, 128))
    lin = Mxfp4Linear(*held)
    lin.tiled = torch.zeros(1280, dtype=torch.uint8)  # (not read: every call below is refused)
    for bad in (torch.zeros(2, 32), torch.zeros(64), torch.zeros(2, 64, dtype=torch.float64), torch.zeros(1, 2, 64)):
        with pytest.raises(ValueError):
            ops.mxfp4_linear(bad, lin)
    with pytest.raises(ValueError):
        ops.mxfp4_linear(held, lin, torch.float64)
    with pytest.raises(RuntimeError):
        ops.mxfp4_linear(bf, lin)


def test_routed_experts_refusals():
    from hibana_amd.kernels import mxfp4_moe
    lib = _lib.lib()
    ok = dict(fc1=256, fc2=256, experts=8, base=0, hidden=256, inter=128, hidden_out=256, gated=1)
    ex = _lib.HbMxfp4Experts(*ok.values())
    need = lib.hb_mxfp4_moe_workspace_bytes(C.byref(ex), 4, 2)
    assert need >= 8 * 256 * 4 and lib.hb_mxfp4_moe_workspace_bytes(None, 4, 2) == 0 and lib.hb_mxfp4_moe_workspace_bytes(C.byref(ex), 0, 2) == 0
    call = lambda **c: lib.hb_mxfp4_moe(*{**dict(ex=C.byref(ex), x=256, ids=256, w=256, m=4, k=2, mode=0, out=256, ws=256, size=need, stream=None), **c}.values())  # noqa: E731
    for c in [dict(ex=None), dict(x=None), dict(ids=None), dict(w=None), dict(out=None), dict(ws=None)]:
        assert call(**c) == _lib.HB_ENULL, c
    for c in [dict(m=0), dict(k=0), dict(mode=3), dict(mode=-1), dict(m=1 << 30), dict(x=264), dict(ids=258), dict(w=257), dict(out=260), dict(ws=264)]:
        assert call(**c) == _lib.HB_EINVAL, c
    assert call(size=need - 1) == _lib.HB_EWORKSPACE
    for c in [dict(hidden=48), dict(inter=80), dict(hidden_out=260), dict(experts=0), dict(base=-1), dict(fc1=264), dict(hidden=0)]:
        bad = _lib.HbMxfp4Experts(*{**ok, **c}.values())
        assert lib.hb_mxfp4_moe_workspace_bytes(C.byref(bad), 4, 2) == 0 and call(ex=C.byref(bad)) == _lib.HB_EINVAL, c
    assert call(ex=C.byref(_lib.HbMxfp4Experts(*{**ok, "fc2": None}.values()))) == _lib.HB_ENULL
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    good = (u8(4, 64, 48), u8(4, 64, 3), u8(4, 96, 16), u8(4, 96, 1))
    held = mxfp4_moe.Mxfp4Experts(*good)
    assert held.gated and held.experts == 4
    for i, t in [(0, u8(4, 64, 40)), (0, u8(4, 80, 48)), (1, u8(4, 64, 5)), (2, u8(3, 96, 16)), (2, u8(4, 96, 32))]:
        with pytest.raises(ValueError):
            mxfp4_moe.Mxfp4Experts(*(t if j == i else g for j, g in enumerate(good)))
    with pytest.raises(ValueError):
        mxfp4_moe.Mxfp4Experts(*good, base=-1)
    x, ids, w = torch.zeros(2, 96, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    held.tiled1 = held.tiled2 = u8(1)  # (not read: every call below is refused)
    for bad in [(x.float(), ids, w), (x[:, :64], ids, w), (x, ids[:1], w), (x, ids, w[:, :2]), (x[0], ids, w)]:
        with pytest.raises(ValueError):
            mxfp4_moe.mxfp4_moe(held, *bad)
    with pytest.raises(RuntimeError):
        mxfp4_moe.mxfp4_moe(held, x, ids, w)  # no CPU path


def test_weights_of_another_format_are_refused():
    from types import SimpleNamespace

    from hibana_amd.kernels import mxfp4_moe
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    other = SimpleNamespace(in_features=64, out_features=32, tiled=torch.zeros(1, dtype=torch.uint8), w3=None, pairs=0)
    with pytest.raises(ValueError):
        ops.mxfp4_linear(x, other)
    with pytest.raises(ValueError):
        mxfp4_moe.mxfp4_moe(SimpleNamespace(shape1=(1, 64, 64), shape2=(1, 64, 64)), x, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))


def test_layouts_that_do_not_fit_their_shapes():
    """Weights handed over in the kernels' layout alone: of the size that the shape has, or refused."""
    from hibana_amd.kernels import mxfp4_moe
    lib = _lib.lib()
    size = lib.hb_mxfp4_tiled_bytes(64, 96)
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    assert Mxfp4Linear(None, None, tiled=u8(size), out_features=64, in_features=96).bytes == 64 * 96 * 17 // 32
    for tiled, n, k in [(None, 64, 96), (u8(size - 1), 64, 96), (u8(size), 96, 96), (u8(size), 0, 0), (u8(size).int(), 64, 96), (u8(2 * size)[::2], 64, 96)]:
        with pytest.raises(ValueError):
            Mxfp4Linear(None, None, tiled=tiled, out_features=n, in_features=k)
    with pytest.raises(ValueError):
        Mxfp4Linear(u8(64, 48), u8(64, 3), tiled=u8(size + 256))
    other = lib.hb_mxfp4_tiled_bytes(96, 32)
    make = lambda a, b, e=4: mxfp4_moe.Mxfp4Experts(None, None, None, None, tiled1=a, tiled2=b, shape1=(e, 64, 96), shape2=(e, 96, 32))  # noqa: E731
    assert make(u8(4, size), u8(4, other)).gated
    for a, b, e in [(None, u8(4, other), 4), (u8(3, size), u8(4, other), 4), (u8(4, size), u8(4, size), 4), (u8(961, size), u8(961, other), 961)]:
        with pytest.raises(ValueError):
            make(a, b, e)


def test_sizes_past_what_a_launch_holds():
    lib = _lib.lib()
    assert lib.hb_mxfp4_tiled_bytes(1 << 28, 256) == 0 and lib.hb_mxfp4_tiled_bytes((1 << 28) - 32, 256) > 0  # 2^32 threads
    assert lib.hb_mxfp4_linear_workspace_bytes(1 << 24, 32, 1 << 13, 0) == 0
    ex = lambda **c: _lib.HbMxfp4Experts(*{**dict(fc1=256, fc2=256, experts=960, base=0, hidden=256, inter=128, hidden_out=256, gated=1), **c}.values())  # noqa: E731
    size = lambda e, m, k: lib.hb_mxfp4_moe_workspace_bytes(C.byref(e), m, k)  # noqa: E731
    assert size(ex(), 4, 2) > 0 and size(ex(experts=961), 4, 2) == 0 and size(ex(), 4, 4097) == 0
    assert size(ex(), 1 << 18, 8) == size(ex(), 1 << 22, 8)  # passes of 2^18 pairs
    assert size(ex(inter=1 << 14), 1 << 20, 8) == size(ex(inter=1 << 14), 1 << 22, 8)  # of what a buffer descriptor reaches
    y = lib.hb_mxfp4_linear(256, None, 0, 4, 256, 64, 128, 264, 0, 256, 1 << 20, None)
    assert y == _lib.HB_EINVAL  # results on 16 bytes
