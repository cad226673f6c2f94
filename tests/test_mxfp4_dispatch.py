"""Which launches a linear in the microscaled four-bit format takes, told by the workspace it asks for (host logic, nothing is launched): none where the
rounding rides in the product's launch, the rounded rows where it goes ahead, their tile layout on the ring."""
import pytest

from hibana_amd import _lib

BF16, MXFP4 = 0, 3


def _way(m, n, k, kind=BF16):
    lib = _lib.lib()
    need = lib.hb_mxfp4_linear_workspace_bytes(m, n, k, kind)
    tiles = (lib.hb_mxfp4_tiled_bytes(m, k) + 255) // 256 * 256
    return {0: "inside", m * k * 17 // 32: "ahead"}.get(need, "ring" if need >= tiles else need)


@pytest.mark.parametrize("m, n, k, way", [
    # at most a tile a compute unit: 80 K values inside
    (1, 5120, 5120, "inside"), (16, 5120, 5120, "inside"), (17, 5120, 5120, "ahead"), (32, 8192, 2560, "inside"), (32, 8192, 2592, "ahead"),
    # two tiles a workgroup: 64 K
    (12, 8224, 5120, "inside"), (13, 8224, 5120, "ahead"), (12, 25600, 5120, "inside"), (13, 25600, 5120, "ahead"), (16, 25600, 5120, "ahead"), (24, 25600, 5120, "ahead"),
    # one tile a workgroup again: 48 K
    (9, 16416, 5120, "inside"), (10, 16416, 5120, "ahead"), (9, 24576, 5120, "inside"), (16, 24576, 5120, "ahead"),
    # past four tiles a compute unit the ring takes what is not inside
    (12, 32768, 5120, "inside"), (16, 32768, 5120, "ahead"), (9, 32800, 5120, "inside"), (10, 32800, 5120, "ring"), (16, 151936, 5120, "ring"),
    # activations that do not fit LDS
    (24, 25600, 5152, "ring"), (31, 25600, 5120, "ring"),
])
def test_rounding_inside_ahead_or_into_tiles(m, n, k, way):
    assert _way(m, n, k) == way


def test_rows_that_come_rounded_need_no_room_below_the_ring():
    assert _way(16, 25600, 5120, MXFP4) == _way(16, 5120, 5120, MXFP4) == "inside" and _way(16, 151936, 5120, MXFP4) == "ring"
