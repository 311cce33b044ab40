"""CPU tests of the host plans of the linears with an end and of the attention on the cache in 4 bits."""

import ctypes
import math
import random

import pytest


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.capi.lib(require_gpu=False)


def test_the_tile_that_is_asked_for(lib):
    splits = ctypes.c_int(7)
    for query in (lib.linear16_tile, lib.f8_linear_tile):
        for bad in ((0, 64, 64, 0), (4, 60, 64, 0), (4, 64, 60, 0), (4, 64, 24, 1), (-1, 64, 64, 0)):
            assert query(*bad, None) == 0 and query(*bad, ctypes.byref(splits)) == 0 and splits.value == 0
        assert query(16, 2560, 2560, 0, None) == 16 and query(1, 2560, 10240, 0, None) == 64 and query(1, 64, 64, 1, None) == 32
    assert lib.linear16_tile(8192, 8192, 8192, 0, ctypes.byref(splits)) == 256256 and splits.value == 1
    assert lib.linear16_tile(238, 5120, 2560, 0, ctypes.byref(splits)) == 64256 and splits.value == 6
    assert lib.f8_linear_tile(238, 5120, 2560, 0, ctypes.byref(splits)) == 48064 and splits.value == 1


def test_workspaces_are_what_the_splits_write(lib):
    rng, splits = random.Random(3), ctypes.c_int()
    divided = 0
    for _ in range(20000):
        M, K, N = (int(math.exp(rng.uniform(0, 9))) for _ in range(3))
        K, N = 16 * min(K, 2048), 64 * min(N, 512)
        for gated in (0, 1):
            part = M * N * 4  # a row's packed columns, whole pieces of 64
            tile = lib.linear16_tile(M, K, N, gated, ctypes.byref(splits))
            want = splits.value * part if splits.value > 1 else 0
            divided += want > 0
            assert tile > 0 and lib.linear16_workspace_bytes(M, K, N, gated) == want
            assert 1 <= splits.value <= 16 and (splits.value == 1 or 4 * splits.value <= -(-K // 64))
            tile = lib.f8_linear_tile(M, K, N, gated, ctypes.byref(splits))
            want = splits.value * part if splits.value > 1 else 0
            assert lib.f8_linear_end_workspace_bytes(M, K, N, gated, 1) == want  # (rows in e4m3 are given)
            if tile >= 1000:  # x in e4m3 by whole blocks, a scale a row and block and 1 KB behind them
                rows, kb = -(-M // 16) * 16, -(-K // 128)
                want += -(-(rows * kb * 132 + 1024) // 256) * 256
            assert lib.f8_linear_end_workspace_bytes(M, K, N, gated, 0) == want
    assert divided > 1000
