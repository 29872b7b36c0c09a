"""Lengths and token counts that do not fit are refused: nothing changes, and the status says so."""
import pytest
import torch

from yapd_b200 import _native as N

pytestmark = pytest.mark.gpu


def dev(*xs, dtype=torch.int32):
    return torch.tensor(xs, dtype=dtype, device="cuda")


def small():
    from yapd_b200.paged import PagedCache
    return PagedCache.empty(1, 12, 4, 1, 32, 4, 3, dtype=torch.float32)


def test_counts_near_the_ends_of_64_bits():
    cache = small()
    cache.reserve(5)
    tables, refs = cache.page_table.clone(), cache.refs.clone()
    most = 2 ** 63 - 1
    for counts in ((most, most - 4, most - 5, most - 7), (most - 2, 8, -1, -most - 1), (2 ** 62, 2 ** 32 + 1, 2 ** 31, 2 ** 33 - 5)):
        assert cache.reserve(dev(*counts, dtype=torch.int64)).tolist() == [False] * 4
        assert cache.status() == N.YAPD_STATUS_BAD_LENGTH
        cache.clear_status()
        assert cache.kv_len.tolist() == [5] * 4
        assert torch.equal(cache.page_table, tables) and torch.equal(cache.refs, refs)
    cache.reserve(dev(7, 0, 1, 3, dtype=torch.int64))
    assert cache.kv_len.tolist() == [12, 5, 6, 8] and cache.status() == 0
    cache.truncate(dev(most, 2, most - 3, 0, dtype=torch.int64))     # all that they have where they have fewer
    assert cache.kv_len.tolist() == [0, 3, 0, 8] and cache.status() == N.YAPD_STATUS_BAD_LENGTH
