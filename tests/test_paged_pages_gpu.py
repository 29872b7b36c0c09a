"""The pages of pools and lists larger than a block of threads, under a window, and captured into graphs."""
import random

import pytest
import torch

from tests.serve_util import Pool
from tests.test_paged_gpu import TYPES, check, make, same

pytestmark = pytest.mark.gpu


def dev(xs, dtype=torch.int32):
    return torch.tensor(xs, dtype=dtype, device="cuda")


def pool_of(slots, pages, ps, columns, seed, dtype=torch.float32):
    from yapd_b200.paged import PagedCache
    kv = torch.randn(1, pages, 2, ps, 1, 32, generator=torch.Generator().manual_seed(seed)).to(dtype)
    cache = PagedCache(kv.cuda(), torch.full((slots, columns), -1, dtype=torch.int32, device="cuda"),
                       torch.zeros(slots, dtype=torch.int64, device="cuda"),
                       torch.zeros(pages, dtype=torch.int32, device="cuda"))
    return cache, Pool(kv, cache.page_table.cpu(), cache.kv_len.cpu(), cache.refs.cpu())


@pytest.mark.parametrize("seed,ps", [(0, 4), (1, 1), (2, 3)])
def test_lists_and_pools_past_a_block_of_threads(seed, ps):
    """2500 slots and 9000 pages: every loop of 1024 threads takes several turns; one page is the tail of many
    listed slots, on both sides of the turns; the pool is full at its low end."""
    r = random.Random(seed)
    slots, pages = 2500, 9000
    cache, pool = pool_of(slots, pages, ps, 7, seed)

    def reserve(adds, some):
        granted = pool.reserve(adds, some)
        assert cache.reserve(dev(adds, torch.int64), dev(some)).tolist() == granted
        same(cache, pool)
        return granted

    first = list(range(0, slots, 5))
    reserve([r.randint(1, 2 * ps) for _ in first], first)
    empty = [s for s in range(slots) if pool.len[s] == 0]
    src = [r.choice(first[:3] + [r.choice(first)]) for _ in empty]      # three requests have hundreds of copies
    cache.fork(dev(src), dev(empty))
    pool.fork(src, empty)
    same(cache, pool)
    every = r.sample(range(slots), slots)
    reserve([r.choice([0, 1, 1, ps]) for _ in every], every)            # their tails are unshared
    some = r.sample(range(slots), 1700)
    takes = [r.randint(0, pool.len[s]) for s in some]
    cache.truncate(dev(takes, torch.int64), dev(some))
    pool.truncate(takes, some)
    same(cache, pool)
    assert cache.compact().tolist() == [pool.compact()]
    same(cache, pool)
    every = r.sample(range(slots), slots)
    reserve([r.randint(0, 2 * ps) for _ in every], every)               # looks past all live pages
    every = r.sample(range(slots), slots)
    granted = reserve([3 * ps] * slots, every)                          # more than there is room for
    assert any(granted) and not all(granted)
    cache.trim(ps, ps, dev(some))
    pool.trim(ps, ps, some)
    same(cache, pool)
    assert cache.compact().tolist() == [pool.compact()]
    same(cache, pool)
    cache.free()
    assert cache.refs.tolist() == [0] * pages and cache.kv_len.tolist() == [0] * slots


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_before_and_after_a_trim(dtype):
    """What a window no longer sees can be given up and overwritten: the attention is the same, bit for bit."""
    cache, q, k, v = make((200, 33, 90, 61), dtype=TYPES[dtype], heads=4, kv_heads=2, T=1, layers=1, ps=8)
    # the trim is for the next token, which stands one further: the last one sees 39 tokens of that window
    want, want_l = cache.attend(0, q.cuda(), window=39, sinks=10, return_lse=True)
    check(cache, q, want, want_l, window=39, sinks=10)
    before = int((cache.refs > 0).sum())
    cache.trim(40, 10)
    assert int((cache.refs > 0).sum()) < before - 10
    cache.kv[:, cache.refs == 0] = float("nan")
    out, lse = cache.attend(0, q.cuda(), window=39, sinks=10, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_l) and bool(torch.isfinite(out).all())
    cache.compact()
    cache.kv[:, cache.refs == 0] = float("nan")
    out, lse = cache.attend(0, q.cuda(), window=39, sinks=10, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_l) and cache.status() == 0


def test_page_operations_in_a_graph():
    """A tick's page operations and attention, captured once and replayed, follow the host model and the eager calls."""
    slots, ps, window, sinks = 9, 4, 13, 3
    cache, pool = pool_of(slots, 90, ps, 12, 5)
    eager, _ = pool_of(slots, 90, ps, 12, 5)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(slots, h, 32, generator=g, device="cuda") for h in (2, 1, 1))
    src, dst, every = dev([0, 2]), dev([7, 8]), list(range(slots))
    granted, live = torch.empty(slots, dtype=torch.bool, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def tick(c):
        c.truncate(1, src)
        c.free(dst)
        c.fork(src, dst)
        granted.copy_(c.reserve(3))
        c.attend(0, q, k, v, window=window, sinks=sinks, out=out)
        c.trim(window, sinks)
        live.copy_(c.compact())

    def model():
        pool.truncate([1, 1], [0, 2])
        pool.truncate([-1, -1], [7, 8])
        pool.fork([0, 2], [7, 8])
        return pool.reserve([3] * slots, every)

    for c in (cache, eager):
        c.reserve(2)
    pool.reserve([2] * slots, every)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tick(eager)                      # the first calls set kernel attributes
    torch.cuda.current_stream().wait_stream(side)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tick(cache)
    for n in range(9):
        graph.replay()
        got, alive, have = granted.tolist(), live.tolist(), out.clone()
        if n:
            tick(eager)
            first = out.clone()
        assert got == model()
        pool.trim(window, sinks, every)
        assert alive == [pool.compact()]
        assert cache.page_table.tolist() == pool.table and cache.kv_len.tolist() == pool.len
        assert cache.refs.tolist() == pool.refs and torch.equal(cache.page_table, eager.page_table)
        assert torch.equal(have, first)
        assert cache.status() == eager.status()
