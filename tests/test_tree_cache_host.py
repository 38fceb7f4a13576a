"""Speculative decoding, host side (no GPU): the cache's checks before a commit,
which caches' rows share memory, and the split rule at its arguments' ends."""

from __future__ import annotations

import itertools
import random

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    from maple_flash_dgx_spark_b200 import _lib
    from maple_flash_dgx_spark_b200.build import build

    build()
    return _lib.lib()


def test_commit_tree_checks_slots_and_counts():
    """Wrong widths and counts are refused before any row moves or any length changes."""
    from maple_flash_dgx_spark_b200.model import KVCache

    cache = KVCache(["full_attention"], None, n_kv=1, head_dim=64, max_len=16, batch=3, dtype=torch.float32, device="cpu")
    path, n = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)

    def refused(path, n, kept=None):
        with pytest.raises(ValueError):
            cache.commit_tree(path, n, kept)
        assert cache.seen == cache.seqlen.tolist() == [0, 0, 0]

    refused(torch.zeros(4, 4, dtype=torch.int32), torch.ones(4, dtype=torch.int32))
    refused(path[0], n)
    refused(path, n[:2])
    refused(path, n, kept=[1, 1])
    refused(path, n, kept=[1, 1, 1, 1])
    refused(path, n, kept=[1, 5, 1])
    refused(path, n, kept=[1, -1, 1])
    with cache.prefill_slot(1):
        refused(path[:2], n[:2])
    cache.tree_slots = {1}
    refused(path, n)
    refused(path[:1], n[:1])
    with cache.prefill_slot(2):
        refused(path[:1], n[:1])


def test_rows_that_share_memory():
    """Against every pair of rows compared, over strides in any order, gaps,
    overlaps by one position and caches in one another's gaps."""
    from maple_flash_dgx_spark_b200.kernels import _rows_overlap

    r, seen = random.Random(3), set()
    for _ in range(4000):
        Bc, n_kv, T, D, es = r.randint(1, 3), r.randint(1, 3), r.randint(1, 3), 8, r.choice([2, 4])
        R = T * D
        strides = [r.choice([0, R - D, R, 2 * R - D, 2 * R, 2 * R + D, 3 * R, 4 * R, 6 * R]) for _ in range(2)]
        ptrs = [4096 + es * r.choice([0, D, R, 2 * R, 3 * R, 6 * R, 9 * R, 40 * R]) for _ in range(r.randint(1, 3))]
        starts = [(p + es * (b * strides[0] + h * strides[1])) for p in ptrs for b in range(Bc) for h in range(n_kv)]
        want = any(abs(x - y) < R * es for x, y in itertools.combinations(starts, 2))
        assert _rows_overlap(ptrs, (Bc, n_kv, T, D), (*strides, D, 1), es) == want
        seen.add((want, len(ptrs) > 1, Bc * n_kv > 1))
    assert len(seen) == 7  # one row of one cache has nothing to overlap with
    assert not _rows_overlap([0], (0, 2, 4, 8), (64, 32, 8, 1), 2)
    # offsets past 32 bits
    assert not _rows_overlap([0, 1 << 40], (64, 8, 1 << 20, 128), (1 << 30, 1 << 27, 128, 1), 2)
    assert _rows_overlap([0, 1 << 33], (64, 8, 1 << 20, 128), (1 << 30, 1 << 27, 128, 1), 2)


@pytest.mark.parametrize("dtype,D", [(1, 64), (1, 128), (1, 256), (0, 128)])
def test_windows_past_every_cache_split_as_none(L, dtype, D):
    """A window no position is outside of leaves the splits as they are, the
    largest number as well."""
    def size(window):
        return L.maple_tree_gqa_workspace_bytes(1, 64, 32, 4, D, 65536, window, dtype)

    assert size(0) > 0
    for window in (65536, 1 << 31, 1 << 62, (1 << 63) - 60, (1 << 63) - 1):
        assert size(window) == size(0), window


def test_narrowing_refuses_before_any_launch(L):
    assert L.maple_narrow_int64(256, 0, 256, None) == 0
    assert L.maple_narrow_int64(256, -1, 256, None) == 1
    assert L.maple_narrow_int64(None, 4, 256, None) == 1
    assert L.maple_narrow_int64(256, 4, None, None) == 1
