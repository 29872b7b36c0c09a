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


@pytest.mark.parametrize("wrong", [13, 2 ** 31, 2 ** 40 + 6, -1, -2 ** 40])
def test_lengths_that_the_tables_do_not_hold(wrong):
    """`kv_len` is the caller's: a slot with a wrong one is empty to attention and left alone by the pages."""
    cache = small()
    cache.reserve(5)
    cache.kv.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q, k, v = (torch.randn(4, 1, 32, device="cuda") for _ in range(3))
    want, want_l = cache.attend(0, q, return_lse=True)
    cache.kv_len[2] = wrong
    kv, tables, refs = cache.kv.clone(), cache.page_table.clone(), cache.refs.clone()

    def status():
        word = cache.status()
        cache.clear_status()
        return word

    out, lse = cache.attend(0, q, return_lse=True)
    assert status() == N.YAPD_STATUS_BAD_LENGTH
    assert bool((out[2] == 0).all()) and bool((lse[2] == -float("inf")).all())
    for b in (0, 1, 3):
        assert torch.equal(out[b], want[b]) and torch.equal(lse[b], want_l[b])
    cache.attend(0, q[2:3], k[2:3], v[2:3], slots=dev(2))
    assert status() == N.YAPD_STATUS_BAD_LENGTH and torch.equal(cache.kv, kv)
    assert cache.reserve(dev(0, 1, 0, 2, dtype=torch.int64)).tolist() == [True, True, False, True]
    assert status() == N.YAPD_STATUS_BAD_LENGTH
    assert cache.kv_len.tolist() == [5, 6, wrong, 7]
    cache.truncate(dev(0, 1, 1, 2, dtype=torch.int64))
    assert status() == N.YAPD_STATUS_BAD_LENGTH
    cache.trim(1)
    assert status() == N.YAPD_STATUS_BAD_LENGTH
    assert cache.kv_len.tolist() == [5, 5, wrong, 5] and torch.equal(cache.page_table[2], tables[2])
    cache.free(dev(1))
    cache.fork(dev(2), dev(1))
    assert status() == N.YAPD_STATUS_BAD_LENGTH
    assert cache.kv_len.tolist() == [5, 0, wrong, 5] and cache.page_table[1].tolist() == [-1] * 3
    assert bool((cache.refs[cache.page_table[2][:2].long()] == 1).all())
    cache.free(dev(2))                       # empties it, whatever its length
    assert status() == N.YAPD_STATUS_BAD_LENGTH
    assert cache.kv_len.tolist() == [5, 0, 0, 5] and cache.page_table[2].tolist() == [-1] * 3
    cache.free()
    assert status() == 0 and cache.refs.tolist() == [0] * 12 and bool((refs >= 0).all())
