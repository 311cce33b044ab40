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


def _divided(n, T, width, H, Hk):
    """Whether keys are divided, at 256 CUs: tables of more than 16 pages, or 32 where the tiles alone give every CU one, and
    tiles below two a CU."""
    G = H // Hk
    rt = 1 if T * G // n <= 64 else 2
    tiles = T * G // (16 * rt)
    return rt, width > (16 if max(tiles, n) * Hk < 256 else 32) and tiles * Hk < 512


def _f32(v):
    return ctypes.c_float(v).value


def test_the_caches_workspace_holds_every_item(lib):
    """What the kernels number on the device, (sequence, tile, chunk of keys), restated: chunks of whole passes of 256 keys, two
    at least and a 256th of the table at least, as spread all over 2,048 / Hk workgroups (256 at most) of a key head."""
    rng = random.Random(5)
    spread = lambda hi: int(hi ** rng.random())  # noqa: E731
    seen = 0
    for _ in range(4000):
        n, Hk, G, d = spread(300), spread(40), spread(32), 8 * rng.randint(1, 16)
        nq = [spread(rng.choice((1, 2, 8, 300))) if rng.random() < 0.9 else 0 for _ in range(n)]
        width = spread(rng.choice((8, 40, 600, 40000)))
        nk = [rng.choice((0, 64 * width, rng.randrange(64 * width + 1), spread(64 * width))) for _ in range(n)]
        T = sum(nq) + rng.choice((0, 0, 5))
        if T == 0:
            continue
        need = lib.cache4_attention_workspace_bytes(n, T, width, Hk * G, Hk, d)
        rt, divided = _divided(n, T, width, Hk * G, Hk)
        assert (need > 0) == divided
        if not divided:
            continue
        seen += 1
        each = Hk * 16 * rt * (8 + 4 * (64 if d <= 64 else 128))
        assert need % each == 0
        items, target = need // each, min(-(-2048 // Hk), 256)
        tiles = [-(-q * G // (16 * rt)) for q in nq]
        passes = 0.0
        for t, k in zip(tiles, nk):
            passes = _f32(passes + _f32(t * -(-k // 256)))
        keys = 256 * max(2, math.ceil(_f32(passes / target)), -(-64 * width // 65536))
        chunks = [max(1, -(-k // keys)) for k in nk]
        assert sum(t * c for t, c in zip(tiles, chunks)) <= items and max(chunks) <= 256
    assert seen > 500


def test_the_caches_memory_beside_16_bits(lib):
    for d, share in ((128, 0.28125), (120, 0.3), (96, 0.375), (80, 0.45), (72, 0.5), (64, 0.28125), (32, 0.5625), (24, 0.75), (16, 1.125), (8, 2.25)):
        assert lib.cache4_bytes(5, 3, d) == share * 5 * 64 * 3 * 2 * d * 2
