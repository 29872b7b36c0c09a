"""Attention over the paged cache, and its pages, against plain implementations."""
import math
import random

import pytest
import torch

from tests.serve_util import Pool, attend64, attend_tolerance
from yapd_b200 import _native as N

pytestmark = pytest.mark.gpu


def make(lens, *, dtype=torch.bfloat16, heads=4, kv_heads=4, D=64, ps=16, T=1, layers=2, spare=3, seed=0,
         page_major=False, fill=float("nan")):
    """A cache whose requests hold `lens` tokens on pages in random order; all that holds no token is `fill`."""
    from yapd_b200.paged import PagedCache
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // ps) for n in lens]
    pages, cols = sum(held) + spare, max(held + [1]) + 1
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    kv = torch.full((layers, pages, 2, ps, kv_heads, D), fill, dtype=dtype)
    at = 0
    for s, n in enumerate(lens):
        for c in range(held[s]):
            page = order[at]
            at += 1
            table[s, c], refs[page] = page, 1
            k = min(ps, n - c * ps)
            kv[:, page, :, :k] = torch.randn(layers, 2, k, kv_heads, D, generator=g).to(dtype)
    q = (1.5 * torch.randn(len(lens), T, heads, D, generator=g)).to(dtype)
    k, v = (torch.randn(len(lens), T, kv_heads, D, generator=g).to(dtype) for _ in range(2))
    dev = kv.cuda()
    if page_major:
        dev = dev.transpose(0, 1).contiguous().transpose(0, 1)
    cache = PagedCache(dev, table.cuda(), torch.tensor(lens, dtype=torch.int64).cuda(), refs.cuda())
    return cache, q, k, v


def tokens(kv, table, layer, s, n, half):
    """Rows of the tokens of slot s, looked up one by one (no page: zeros, for tokens that nothing sees)."""
    ps = kv.shape[3]
    zero = torch.zeros(kv.shape[4:], dtype=kv.dtype)
    rows = [kv[layer, table[s][j // ps], half, j % ps] if table[s][j // ps] >= 0 else zero for j in range(n)]
    return torch.stack(rows) if rows else torch.zeros(0, *kv.shape[4:], dtype=kv.dtype)


def check(cache, q, out, lse, *, layer=0, slots=None, causal=True, window=0, sinks=0, scale=None):
    kv, table, lens = cache.kv.cpu(), cache.page_table.tolist(), cache.kv_len.tolist()
    D, worst = q.shape[-1], 0.0
    scale = D ** -0.5 if scale is None else scale
    for b in range(q.shape[0]):
        s = b if slots is None else slots[b]
        n = lens[s]
        want = attend64(tokens(kv, table, layer, s, n, 0), tokens(kv, table, layer, s, n, 1), q[b], n,
                        causal=causal, window=window, sinks=sinks, scale=scale)
        o, l, size, prod = want
        tol_o, tol_l = attend_tolerance(q.dtype, o, size, prod, n, D)
        empty = l == -math.inf
        got_l = lse[b].cpu().double()
        assert torch.equal(got_l == -math.inf, empty)
        err = (out[b].cpu().double() - o).abs()
        assert bool((err <= tol_o).all()), (b, n, float((err / tol_o).max()))
        dl = (got_l - l).abs()[~empty]
        assert bool((dl <= tol_l[~empty]).all()), (b, n, float((dl / tol_l[~empty]).max()))
        worst = max(worst, float((err / tol_o).max()) if err.numel() else 0.0)
    return worst


CASES = [
    # dtype, heads, kv_heads, D, page size, T, causal, window, sinks, lens
    ("bf16", 4, 4, 64, 16, 1, True, 0, 0, (1, 2, 15, 16, 17, 100)),
    ("bf16", 16, 16, 64, 16, 1, True, 0, 0, (417, 0, 33)),
    ("f16", 8, 2, 128, 64, 1, True, 0, 0, (300, 64, 65, 1)),
    ("f32", 4, 4, 64, 16, 1, True, 0, 0, (1, 31, 129)),
    ("f32", 6, 2, 96, 5, 7, True, 0, 0, (7, 8, 40, 93)),
    ("f32", 8, 1, 128, 16, 32, False, 0, 0, (32, 50)),
    ("f32", 3, 3, 32, 7, 2, True, 20, 3, (2, 19, 30, 120)),
    ("bf16", 3, 3, 32, 7, 2, True, 20, 3, (2, 19, 30, 120)),
    ("bf16", 4, 4, 64, 16, 16, False, 0, 0, (16, 17, 90, 200)),
    ("bf16", 4, 4, 64, 16, 32, True, 0, 0, (32, 33, 250)),
    ("f16", 12, 3, 96, 16, 5, True, 0, 0, (5, 64, 161)),
    ("bf16", 32, 4, 64, 16, 16, True, 0, 0, (16, 70, 140)),
    ("f16", 8, 1, 128, 1, 32, False, 0, 0, (32, 64, 95)),
    ("bf16", 16, 4, 128, 16, 1, True, 64, 10, (5, 63, 64, 65, 75, 76, 400)),
    ("bf16", 4, 2, 64, 100, 3, True, 1, 0, (3, 99, 100, 101, 350)),
    ("f16", 4, 4, 64, 8, 16, False, 9, 40, (16, 30, 60, 128)),
    ("f16", 4, 4, 64, 16, 1, False, 300, 0, (10, 299, 300, 301, 500)),
    ("bf16", 2, 1, 32, 3, 4, True, 16, 1000, (4, 50, 90)),
]
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.mark.parametrize("dtype,heads,kv_heads,D,ps,T,causal,window,sinks,lens", CASES)
def test_attend(dtype, heads, kv_heads, D, ps, T, causal, window, sinks, lens):
    cache, q, k, v = make(lens, dtype=TYPES[dtype], heads=heads, kv_heads=kv_heads, D=D, ps=ps, T=T, seed=len(lens) + T)
    # the new tokens' pages must have room, whatever the length
    out, lse = cache.attend(1, q.cuda(), k.cuda(), v.cuda(), causal=causal, window=window, sinks=sinks, return_lse=True)
    check(cache, q, out, lse, layer=1, causal=causal, window=window, sinks=sinks)
    again, lse2 = cache.attend(1, q.cuda(), causal=causal, window=window, sinks=sinks, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)   # the rows are where they were stored
    short = any(n < T for n in lens)
    assert cache.status() == (N.YAPD_STATUS_BAD_LENGTH if short else 0)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attend_long_split(dtype):
    """One long request among short and empty ones: its keys are shared out and joined."""
    lens = [5000, 0, 3, 700] + [0] * 40 + [1] * 5
    cache, q, k, v = make(lens, dtype=TYPES[dtype], heads=4, kv_heads=2, D=64, T=1, layers=1)
    out, lse = cache.attend(0, q.cuda(), return_lse=True)
    check(cache, q, out, lse)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


def test_attend_many_requests():
    r = random.Random(4)
    lens = [r.choice([0, 1, 2, 16, 17, r.randint(1, 60)]) for _ in range(700)]
    cache, q, k, v = make(lens, heads=2, kv_heads=1, D=32, ps=4, layers=1)
    out, lse = cache.attend(0, q.cuda(), return_lse=True)
    check(cache, q, out, lse)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_only_the_new_rows_are_stored(dtype):
    cache, q, k, v = make((5, 37, 64), dtype=TYPES[dtype], T=5)
    before = cache.kv.clone()
    cache.attend(1, q.cuda(), k.cuda(), v.cuda())
    ps = 16
    for b, n in enumerate((5, 37, 64)):
        for i in range(5):
            t = n - 5 + i
            page = int(cache.page_table[b, t // ps])
            for half, rows in ((0, k), (1, v)):
                assert torch.equal(cache.kv[1, page, half, t % ps].cpu(), rows[b, i])
                before[1, page, half, t % ps] = rows[b, i].cuda()
    assert torch.equal(cache.kv.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), "lowest"])
def test_masked_places_do_not_matter(dtype, bad):
    """NaN, infinities and the type's lowest value where no query, or only a later one, sees them."""
    dt = TYPES[dtype]
    value = torch.finfo(dt).min if bad == "lowest" else bad
    T, n, window, sinks = 4, 77, 20, 6
    cache, q, k, v = make((n,), dtype=dt, T=T, layers=1, ps=8, fill=value)
    kv, table = cache.kv, cache.page_table[0].tolist()
    for j in range(sinks, n - T - window + 1):       # hidden from every query
        kv[0, table[j // 8], :, j % 8] = value
    out, lse = cache.attend(0, q.cuda(), window=window, sinks=sinks, return_lse=True)
    assert bool(torch.isfinite(out).all())
    clean = kv.clone()
    for j in range(sinks, n - T - window + 1):
        clean[0, table[j // 8], :, j % 8] = 0.0
    cache.kv.copy_(clean)
    want, want_l = cache.attend(0, q.cuda(), window=window, sinks=sinks, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_l)
    # the last token's value row: the queries before it do not see it, the last one does
    j = n - 1
    kv[0, table[j // 8], 1, j % 8] = value
    out, lse = cache.attend(0, q.cuda(), window=window, sinks=sinks, return_lse=True)
    assert torch.equal(out[:, :-1], want[:, :-1]) and torch.equal(lse, want_l)
    assert bad == "lowest" or not bool(torch.isfinite(out[:, -1]).any())
    # and so for its key row
    kv[0, table[j // 8], 1, j % 8] = 0.0
    kv[0, table[j // 8], 0, j % 8] = value
    out, lse = cache.attend(0, q.cuda(), window=window, sinks=sinks, return_lse=True)
    assert torch.equal(out[:, :-1], want[:, :-1]) and torch.equal(lse[:, :-1], want_l[:, :-1])


def test_large_scores():
    """Scores far apart, and in the thousands: the running maximum carries the sum."""
    for dt in TYPES.values():
        cache, q, k, v = make((130,), dtype=dt, layers=1)
        q = q * 40
        out, lse = cache.attend(0, q.cuda(), scale=1.0, return_lse=True)
        check(cache, q, out, lse, scale=1.0)
        # every score -inf: nothing is seen
        cache.kv[:, :, 0] = -1.0
        q = torch.full_like(q, torch.finfo(dt).max)
        out, lse = cache.attend(0, q.cuda(), scale=float("inf") if dt != torch.float32 else 1.0, return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_strides_slots_layouts_and_streams():
    """Rows sliced from a fused projection, a page-major pool, permuted slots, another stream."""
    lens = (40, 7, 0, 129, 16)
    cache, q, k, v = make(lens, heads=8, kv_heads=2, T=3, page_major=True)
    plain = (q, k, v)
    fused = torch.randn(4, 3, 8 + 2 + 2, 64).to(torch.bfloat16)
    slots = [3, 0, 4, 1]
    for b, s in enumerate(slots):
        fused[b, :, :8], fused[b, :, 8:10], fused[b, :, 10:] = (t[s] for t in plain)
    dev = fused.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    wide = torch.zeros(4, 3, 8, 128, dtype=torch.bfloat16, device="cuda")
    with torch.cuda.stream(side):
        out, lse = cache.attend(1, dev[:, :, :8], dev[:, :, 8:10], dev[:, :, 10:],
                                slots=torch.tensor(slots, dtype=torch.int32, device="cuda"),
                                out=wide[..., :64], return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    check(cache, fused[:, :, :8], out, lse, layer=1, slots=slots)
    assert bool((wide[..., 64:] == 0).all())
    # rows that are not 16-byte aligned, and a head dimension with a stride, are read from a copy
    odd = torch.zeros(4, 3, 8, 65, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = dev[:, :, :8]
    again = cache.attend(1, odd[..., 1:], slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    turned = dev[:, :, :8].transpose(2, 3).contiguous().transpose(2, 3)
    third = cache.attend(1, turned, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    assert torch.equal(again, out) and torch.equal(third, out)
    one = cache.attend(1, dev[:, -1, :8], slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    assert one.shape == (4, 8, 64) and torch.equal(one, out[:, -1])


def test_offsets_past_32_bits():
    """Pages more than 2^32 elements into the pool."""
    from yapd_b200.paged import PagedCache
    block = 2 * 16 * 16 * 64
    pages = 2 ** 32 // block + 40
    kv = torch.empty(1, pages, 2, 16, 16, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[pages - 1, 3, pages - 7], [pages // 2 + 1, pages - 2, -1]], dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    kv[0, table[table >= 0].long()] = torch.randn(5, 2, 16, 16, 64, device="cuda").to(torch.bfloat16)
    cache = PagedCache(kv, table, torch.tensor([44, 20], device="cuda"), refs)
    q, k, v = (torch.randn(2, 1, 16, 64).to(torch.bfloat16) for _ in range(3))
    out, lse = cache.attend(0, q.cuda(), k.cuda(), v.cuda(), return_lse=True)
    small = cache.kv[:, table[table >= 0].long()].cpu()
    for b, (ids, n) in enumerate((([0, 1, 2], 44), ([3, 4], 20))):
        rows = small[0, ids].transpose(0, 1).reshape(2, -1, 16, 64)[:, :n]
        o, l, size, prod = attend64(rows[0], rows[1], q[b], n, causal=True, window=0, sinks=0, scale=0.125)
        tol_o, tol_l = attend_tolerance(torch.bfloat16, o, size, prod, n, 64)
        assert bool(((out[b].cpu().double() - o).abs() <= tol_o).all())
    cache.compact()
    assert torch.equal(cache.kv[0, cache.page_table[cache.page_table >= 0].long()].cpu(), small[0])


def test_bad_tables_are_reported():
    cache, q, k, v = make((40, 40), layers=1, fill=0.0)
    cache.page_table[0, 1] = 10 ** 6
    cache.page_table[1, 0] = -1
    out, lse = cache.attend(0, q.cuda(), return_lse=True)
    assert cache.status() == N.YAPD_STATUS_BAD_PAGE
    assert bool(torch.isfinite(out).all())
    cache.clear_status()
    cache.page_table[1, 2] = -1
    cache.page_table[0, 1] = 0
    cache.page_table[1, 0] = 0
    cache.attend(0, q.cuda(), k.cuda(), v.cuda())
    assert cache.status() == N.YAPD_STATUS_BAD_PAGE
    cache.clear_status()
    cache.attend(0, q.cuda(), slots=torch.tensor([7, -1], dtype=torch.int32, device="cuda"))
    cache.attend(0, q.cuda(), k.cuda(), v.cuda(), slots=torch.tensor([7, -1], dtype=torch.int32, device="cuda"))
    assert cache.status() == N.YAPD_STATUS_BAD_SLOT


def test_shared_pages_are_not_written():
    cache, q, k, v = make((20, 0), layers=1)
    cache.fork(torch.tensor([0], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda"))
    before = cache.kv.clone()
    cache.attend(0, q.cuda(), k.cuda(), v.cuda())
    assert cache.status() == N.YAPD_STATUS_SHARED_PAGE
    assert torch.equal(cache.kv.view(torch.int16), before.view(torch.int16))


# ------------------------------------------------------------------------ pages

def same(cache, pool):
    assert cache.page_table.tolist() == pool.table
    assert cache.kv_len.tolist() == pool.len
    assert cache.refs.tolist() == pool.refs
    kv = cache.kv.cpu()
    assert torch.equal(kv.contiguous().view(torch.uint8), pool.kv.contiguous().view(torch.uint8))


@pytest.mark.parametrize("seed,ps,slots,dtype", [(0, 16, 12, "bf16"), (1, 1, 6, "f32"), (2, 5, 40, "f16"), (3, 8, 3, "bf16")])
def test_pages_follow_the_host_model(seed, ps, slots, dtype):
    r = random.Random(seed)
    from yapd_b200.paged import PagedCache
    pages = slots * 4 + 5
    kv = torch.randn(3, pages, 2, ps, 2, 32, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype])
    cache = PagedCache(kv.cuda(), torch.full((slots, 9), -1, dtype=torch.int32, device="cuda"),
                       torch.zeros(slots, dtype=torch.int64, device="cuda"),
                       torch.zeros(pages, dtype=torch.int32, device="cuda"))
    pool = Pool(kv, cache.page_table.cpu(), cache.kv_len.cpu(), cache.refs.cpu())
    dev = lambda xs, dt=torch.int32: torch.tensor(xs, dtype=dt, device="cuda")  # noqa: E731
    forked = 0
    for step in range(120):
        op = r.choice(["reserve", "reserve", "reserve", "fork", "fork", "truncate", "free", "trim", "compact"])
        some = r.sample(range(slots), r.randint(1, slots))
        if op == "reserve":
            adds = [r.choice([0, 1, 2, ps, r.randint(0, 3 * ps)]) for _ in some]
            if r.random() < 0.3:
                adds, some = [adds[0]] * slots, list(range(slots))
                got = cache.reserve(adds[0])
            else:
                got = cache.reserve(dev(adds, torch.int64), dev(some))
            assert got.tolist() == pool.reserve(adds, some)
        elif op == "fork":
            empty = [s for s in range(slots) if pool.len[s] == 0]
            full = [s for s in range(slots) if pool.len[s]]
            if not empty or not full:
                continue
            src = [r.choice(full) for _ in empty]
            cache.fork(dev(src), dev(empty))
            pool.fork(src, empty)
            forked += 1
        elif op == "truncate":
            takes = [r.randint(0, pool.len[s]) for s in some]
            cache.truncate(dev(takes, torch.int64), dev(some))
            pool.truncate(takes, some)
        elif op == "free":
            some = some[: max(1, slots // 4)]
            cache.free(dev(some))
            pool.truncate([-1] * len(some), some)
        elif op == "trim":
            window, sinks = r.randint(1, 4 * ps), r.randint(0, 2 * ps)
            cache.trim(window, sinks, dev(some))
            pool.trim(window, sinks, some)
        else:
            assert cache.compact().tolist() == [pool.compact()]
        same(cache, pool)
    assert forked
    cache.free()
    assert cache.refs.tolist() == [0] * pages


def test_pages_refusals_on_the_device():
    from yapd_b200.paged import PagedCache
    cache = PagedCache.empty(1, 4, 4, 1, 32, 6, 3, dtype=torch.float32)
    dev = lambda *xs: torch.tensor(xs, dtype=torch.int32, device="cuda")  # noqa: E731
    assert cache.reserve(5, dev(0, 0, 9, -3, 1)).tolist() == [True, False, False, False, True]
    assert cache.status() == N.YAPD_STATUS_BAD_SLOT
    assert cache.kv_len.tolist() == [5, 5, 0, 0, 0, 0]
    cache.clear_status()
    assert cache.reserve(1, dev(2, 3)).tolist() == [False, False]
    assert cache.status() == N.YAPD_STATUS_OUT_OF_PAGES
    cache.clear_status()
    assert cache.reserve(8, dev(0)).tolist() == [False]          # twelve tokens are all that its table holds
    assert cache.status() == N.YAPD_STATUS_BAD_LENGTH
    cache.clear_status()
    cache.fork(dev(0, 0, 2, 0), dev(1, 2, 4, 2))   # not empty, fine, a target itself, listed twice
    assert cache.status() == N.YAPD_STATUS_BAD_SLOT
    assert cache.kv_len.tolist() == [5, 5, 5, 0, 0, 0] and cache.refs.tolist() == [2, 2, 1, 1]
    cache.clear_status()
    cache.truncate(6, dev(1))
    assert cache.status() == N.YAPD_STATUS_BAD_LENGTH and cache.kv_len.tolist() == [5, 0, 5, 0, 0, 0]
    cache.clear_status()
    cache.free(dev(0, 0, 2))
    assert cache.status() == N.YAPD_STATUS_BAD_SLOT and cache.refs.tolist() == [0, 0, 0, 0]
    cache.clear_status()
    cache.copy_pages(dev(0, 7), dev(1, 2))
    assert cache.status() == N.YAPD_STATUS_BAD_PAGE


@pytest.mark.parametrize("page_major", [False, True])
def test_copy_pages(page_major):
    cache, *_ = make((64, 64, 64), layers=3, fill=0.0, page_major=page_major)
    want = cache.kv.cpu().clone()
    src, dst = [0, 5, 3], [7, 1, 2]
    want[:, dst] = want[:, src]
    cache.copy_pages(torch.tensor(src, dtype=torch.int32, device="cuda"),
                     torch.tensor(dst, dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.kv.cpu(), want) and cache.status() == 0


def test_window_reads_no_trimmed_page():
    """Attention with a window is the same before and after the pages that it does not see are given up."""
    cache, q, k, v = make((200, 33, 90), T=1, layers=1, ps=8)
    want = cache.attend(0, q.cuda(), window=40, sinks=10)
    # the next query stands one further: give up what it will not see, then let it in
    cache.trim(40, 10)
    cache.kv[:, cache.refs == 0] = float("nan")
    assert int((cache.page_table == -1).sum()) > 10
    assert torch.equal(cache.attend(0, q.cuda(), window=39, sinks=10), cache.attend(0, q.cuda(), window=39, sinks=10))
    cache.reserve(1)
    out, lse = cache.attend(0, q.cuda(), k.cuda(), v.cuda(), window=40, sinks=10, return_lse=True)
    check(cache, q, out, lse, window=40, sinks=10)
    assert cache.status() == 0 and want.shape == out.shape


@pytest.mark.parametrize("dtype", list(TYPES))
def test_expired_waits_are_reported_and_contained(dtype):
    """Waits that give up at once: the status says so, and the next call is exact again."""
    lens = [3000, 5, 700, 0, 64]
    cache, q, k, v = make(lens, dtype=TYPES[dtype], heads=4, kv_heads=2, layers=1)
    want, want_l = cache.attend(0, q.cuda(), return_lse=True)
    for _ in range(3):
        cache.attend(0, q.cuda(), wait_limit_ns=-1)
        assert cache.status() == N.YAPD_STATUS_WAIT_TIMEOUT
        cache.clear_status()
        out, lse = cache.attend(0, q.cuda(), return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_l) and cache.status() == 0


def test_graph_capture_and_repeats():
    """A tick captured into a graph gives the eager call's results, whatever ran between."""
    lens = [100, 1, 900] + [33] * 60
    cache, q, k, v = make(lens, heads=4, kv_heads=4, layers=1)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    want = cache.attend(0, q, k, v)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        cache.attend(0, q, k, v, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert cache.status() == 0


def test_example_runs():
    """The example's beams share pages, stay within the window's pages, and are scored consistently."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    a, la, cache = m.run(requests=3, beams=2, prompt=40, tokens=30)
    b, lb, _ = m.run(requests=3, beams=2, prompt=40, tokens=30)
    assert torch.equal(a, b) and torch.equal(la, lb)         # the same seed, the same tokens
    assert cache.status() == 0 and bool(torch.isfinite(la).all()) and bool((la < 0).all())
    live = int((cache.refs > 0).sum())
    assert live == int((cache.page_table >= 0).sum()) and bool((cache.refs[:live] == 1).all())
    # a single candidate needs no fork
    one, l1, _ = m.run(requests=3, beams=1, prompt=40, tokens=30)
    assert one.shape == a.shape
