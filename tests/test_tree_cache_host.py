"""Speculative decoding, host side (no GPU): the cache's checks before a commit."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


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
