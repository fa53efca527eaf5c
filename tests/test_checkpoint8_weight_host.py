"""The weight gradient's plans, on a host without a GPU (148 SMs are taken where there is no device)."""
import ctypes as C

import pytest


def plan(native, rows, n, k):
    p = (C.c_int32 * 3)(-1, -1, -1)
    return native.lib.bsrl_linear8_wgrad_plan(rows, n, k, p), list(p)


@pytest.mark.parametrize("rows,n,k", [(0, 8, 8), (-1, 8, 8), (2 ** 31 - 256, 8, 8), (4, 0, 8), (4, 8, 0), (4, 2 ** 20 + 1, 8), (4, 2 ** 20, 2049)])
def test_plan_refuses(native, rows, n, k):
    assert plan(native, rows, n, k) == (-2, [-1, -1, -1])
    assert native.last_error().startswith("linear8_wgrad_plan")


def test_plan_needs_room(native):
    assert native.lib.bsrl_linear8_wgrad_plan(4, 8, 8, None) == -1


def test_plans_fit_their_sizes_and_workspaces(native):
    """Tiles that cover the weight, pieces that hold at least a stage, and room for every piece's partial tiles; all three forms occur."""
    forms = set()
    for rows in (1, 64, 65, 1856, 20994, 100003, 475136, 2 ** 31 - 257):
        for n, k in ((1, 1), (64, 64), (200, 671), (1024, 256), (1985, 10), (1916, 432), (2048, 2048), (2 ** 20, 8), (8, 2 ** 20)):
            rc, (tile_n, tile_k, pieces) = plan(native, rows, n, k)
            stages = -(-rows // 64)
            assert rc == 0 and tile_n in (128, 256, 512) and tile_k % 32 == 0 and 0 < tile_k <= 256 and 1 <= pieces <= min(stages, 2 * 148)
            if tile_n > 128:
                assert tile_k % 64 == 0                         # half of the tile per CTA
            padded = -(-n // tile_n) * tile_n * -(-k // tile_k) * tile_k
            assert native.lib.bsrl_linear8_wgrad_workspace_bytes(rows, n, k, 1) >= padded * pieces * 4
            forms.add(tile_n)
    assert forms == {128, 256, 512}
