"""CPU tests of the packed operators' host plans over sizes of every kind, no keys and no rows among them."""

import ctypes
import random

import pytest


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.capi.lib(require_gpu=False)


@pytest.mark.parametrize("rows", [1, 15, 16, 64, 128, 4096, 100000])
@pytest.mark.parametrize("n", [1, 3, 64, 200])
def test_attention_without_any_keys_needs_no_workspace(lib, rows, n):
    # a division by a chunk of no keys ended the process here from 16 rows a sequence on
    for H, Hk, d in ((4, 4, 64), (32, 8, 128), (1, 1, 8)):
        assert lib.packed_attention_workspace_bytes(n, rows, 0, H, Hk, d) == 0


def test_scales_that_pass_fp32_in_the_exponent_are_refused(lib):
    # (scale log2(e) was infinite in the kernel, and every row NaN)
    p, cu = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 20)
    for scale, rc in ((3e38, -2), (2.4e38, -2), (float("inf"), -2), (1e38, -1)):  # (-1: the next check, of q)
        got = lib.packed_attention(None, p, p, p, 256, 64, 256, 64, 256, 64, 256, 64, cu, cu, 2, 8, 8, 4, 2, 64, 0, scale, 0,
                                   None, 0, None)
        assert got == rc, scale


def test_attention_workspace_over_all_sizes(lib):
    rng = random.Random(0)
    spread = lambda hi: int(hi ** rng.random()) - 1  # noqa: E731  (0 among them)
    for _ in range(20000):
        n, Tq, Tk, Hk, G = 1 + spread(4000), spread(1 << 20), spread(1 << 24), 1 + spread(64), 1 + spread(64)
        d = 8 * rng.randint(1, 16)
        need = lib.packed_attention_workspace_bytes(n, Tq, Tk, Hk * G, Hk, d)
        if need:  # m, l and O of every row and chunk, at most 256 chunks
            rows = Tq * Hk * G
            assert need % 4 == 0 and 2 * rows * (8 + 4 * d) <= need <= 256 * rows * (8 + 4 * d) + 256


def test_f8_workspace_over_all_sizes(lib):
    rng = random.Random(1)
    spread = lambda hi: int(hi ** rng.random()) - 1  # noqa: E731
    for _ in range(20000):
        M, K, N = spread(1 << 16), 16 * (1 + spread(2048)), 8 * (1 + spread(4096))
        need, parts = lib.f8_linear_workspace_bytes(M, K, N), lib.f8_linear_partials_bytes(M, K, N)
        assert parts % (4 * max(M * N, 1)) == 0 and (parts > 0) == (M > 0)
        if M <= 16:
            assert need == 0
        else:  # x in e4m3 by whole blocks, and a scale for each row's block
            rows, kb = (M + 15) // 16 * 16, (K + 127) // 128
            assert need >= rows * kb * 132
