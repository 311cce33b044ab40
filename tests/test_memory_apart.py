"""Whether two views share memory (the check behind every ``out=``), against a count of their bytes; on the CPU."""

import random

import pytest
import torch


def _bytes(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s * t.element_size()
    at = t.data_ptr() + at.flatten()
    return set((at[:, None] + torch.arange(t.element_size())).flatten().tolist())


def _share(K, a, b):
    try:
        K._apart("here", "out", a, b)
    except Exception as e:  # noqa: BLE001
        assert e.code == -3
        return True
    return False


def test_views_of_one_buffer(pkg):
    K, rng = pkg.kernels, random.Random(0)
    buf = torch.zeros(4000, dtype=torch.uint8)
    met = 0

    def view():
        size, dims = rng.choice((1, 2, 4)), rng.randrange(1, 4)
        t = buf.view((torch.uint8, torch.float16, None, torch.float32)[size - 1])
        shape = [rng.choice((0, 1, 2, 3, 5, 8)) if rng.random() < 0.9 else 1 for _ in range(dims)]
        if rng.random() < 0.5:  # rows of one width, parts of a row
            stride = [rng.choice((24, 48, 60)), rng.choice((1, 4, 8, 12)), 1][3 - dims:]
        else:
            stride = [rng.randrange(0, 40) for _ in range(dims)]
        return t.as_strided(shape, stride, rng.randrange(0, 200))

    for _ in range(6000):
        a, b = view(), view()
        want = bool(_bytes(a) & _bytes(b))
        met += want
        assert _share(K, a, b) == want == _share(K, b, a), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert 300 < met < 5700  # (either happens often)


def test_parts_of_wide_rows(pkg):
    K = pkg.kernels
    wide = torch.zeros(1 << 14, 24, 64, dtype=torch.float16)
    q, k, v = wide[:, :8], wide[:, 8:16], wide[:, 16:]
    for a in (q, k, v):
        for b in (q, k, v):
            assert _share(K, a, b) == (a is b)
    assert not _share(K, wide[:, 0::2], wide[:, 1::2]) and not _share(K, wide[0::2], wide[1::2]) and _share(K, wide[0::2], wide[1::3])
    assert _share(K, q[1:], q[:-1]) and _share(K, q[..., 32:], q[..., :40]) and not _share(K, q[..., 32:], q[..., :32])
    assert not _share(K, wide[:100], wide[100:]) and _share(K, wide[:101], wide[100:])
    rows = wide.view(1 << 14, -1)
    assert not _share(K, rows[:, :640], rows[:, 640:1280].unflatten(1, (10, 64))) and _share(K, rows[:1].expand(7, -1), rows[0, 3:4])
    with pytest.raises(pkg.capi.EsmError) as e:
        K._apart("here", "out", rows[1:], None, wide[:0], rows[:-1])
    assert e.value.code == -3
    K._apart("here", "out", rows[:0], rows)
