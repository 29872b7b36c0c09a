"""Attention over the paged cache where its arithmetic is at its ends."""
import math

import pytest
import torch

from tests.test_paged_gpu import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads,T,window,sinks", [(4, 4, 1, 0, 0), (8, 2, 1, 300, 20), (8, 4, 3, 0, 0), (8, 2, 16, 0, 0),
                                                           (8, 1, 5, 200, 33)])
@pytest.mark.parametrize("gap", [8, 12, 15, 17, 18, 20, 22])
def test_small_weights_under_large_ones(dtype, heads, kv_heads, T, window, sinks, gap):
    """Tokens with a value of 0 take the mass; all others, `gap` nats below, have large values of one sign:
    the output is what the small weights add up to."""
    cache, q, k, v = make((500, 161), dtype=TYPES[dtype], heads=heads, kv_heads=kv_heads, T=T, layers=1, fill=0.0)
    kv, table = cache.kv, cache.page_table.tolist()
    kv *= 0.05
    kv[..., 0, :, :, 0] = 0.0
    kv[:, :, 1] = 1000.0 + 2000.0 * kv[:, :, 1]
    q[..., 1:] *= 0.1
    q[..., 0] = 8.0
    for s, n in enumerate((500, 161)):
        for j in range(0, n, 16):            # the first one of them among the first tokens
            kv[0, table[s][j // 16], 0, j % 16, :, 0] = gap
            kv[0, table[s][j // 16], 1, j % 16] = 0.0
    out, lse = cache.attend(0, q.cuda(), window=window, sinks=sinks, return_lse=True)
    check(cache, q, out, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, -1.5, 1e-44, 2.0])
@pytest.mark.parametrize("heads,kv_heads,T,causal,window,sinks", [(4, 4, 1, True, 0, 0), (8, 2, 5, True, 0, 0), (8, 4, 2, False, 0, 0),
                                                                  (8, 1, 3, True, 30, 7), (4, 2, 16, False, 20, 3)])
def test_scales(dtype, scale, heads, kv_heads, T, causal, window, sinks):
    """A scale of 0 gives the mean of what is seen; a negative one turns the order of the scores."""
    cache, q, k, v = make((16, 29, 64, 333), dtype=TYPES[dtype], heads=heads, kv_heads=kv_heads, T=T, layers=1)
    mask = dict(causal=causal, window=window, sinks=sinks)
    out, lse = cache.attend(0, q.cuda(), scale=scale, return_lse=True, **mask)
    if scale < 0:       # the bounds go by the products' sizes: the same attention of the negative queries
        check(cache, -q, out, lse, scale=-scale, **mask)
    else:
        check(cache, q, out, lse, scale=scale, **mask)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads,T,causal,window,sinks", [(4, 4, 1, True, 0, 0), (8, 2, 1, True, 0, 0), (8, 4, 3, True, 0, 0),
                                                                  (8, 1, 1, False, 0, 0), (8, 2, 16, False, 0, 0), (6, 3, 2, True, 90, 5)])
@pytest.mark.parametrize("j,score", [(0, 0), (2, 30), (40, 3), (77, -10), (100, 40), (150, -22), (199, 0), (199, 25), (160, -60)])
def test_infinite_values_that_are_seen(dtype, heads, kv_heads, T, causal, window, sinks, j, score):
    """A value that is infinite makes the output infinite wherever its tile lies, for the rows that see it and
    whatever its weight; values of both signs and NaN make it NaN; the other dims do not change."""
    n = 200
    cache, q, k, v = make((n, 33), dtype=TYPES[dtype], heads=heads, kv_heads=kv_heads, T=T, layers=1, fill=0.0, seed=j)
    kv, row = cache.kv, cache.page_table[0].tolist()
    q[..., 0] = 8.0
    kv[0, :, 0, :, :, 0] = 0.0
    kv[0, row[j // 16], 0, j % 16, :, 0] = score          # 64^-0.5 * 8 = 1
    mask = dict(causal=causal, window=window, sinks=sinks)
    want, want_l = cache.attend(0, q.cuda(), return_lse=True, **mask)
    inf = float("inf")
    kv[0, row[j // 16], 1, j % 16, :, 3] = inf
    kv[0, row[j // 16], 1, j % 16, :, 17] = -inf
    kv[0, row[j // 16], 1, j % 16, :, 40] = float("nan")
    kv[0, row[j // 16], 1, j % 16, :, 63] = inf
    kv[0, row[n // 2 // 16], 1, n // 2 % 16, :, 63] = -inf if j != n // 2 else float("nan")
    out, lse = cache.attend(0, q.cuda(), return_lse=True, **mask)
    assert torch.equal(lse, want_l)
    for i in range(T):
        p = n - T + i
        sees = lambda t: (not causal or t <= p) and (not window or t > p - window or t < sinks)  # noqa: E731
        if sees(j):
            assert bool((out[0, i, :, 3] == inf).all()) and bool((out[0, i, :, 17] == -inf).all())
            assert bool(out[0, i, :, 40].isnan().all())
        if sees(j) and sees(n // 2):
            assert bool(out[0, i, :, 63].isnan().all())
        rest = [d for d in range(64) if d not in ((3, 17, 40, 63) if sees(j) else (63,) if sees(n // 2) else ())]
        assert torch.equal(out[0, i][:, rest], want[0, i][:, rest])
    assert torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ps,T", [(16, 1), (100, 1), (7, 12), (64, 32)])
def test_infinite_values_of_long_requests(dtype, ps, T):
    """The same where a request is cut and joined; NaN scores stay NaN."""
    n, inf = 9000, float("inf")
    cache, q, k, v = make((n, 700), dtype=TYPES[dtype], heads=8, kv_heads=4, T=T, layers=1, ps=ps, fill=0.0)
    kv, table = cache.kv, cache.page_table.tolist()
    for j, d in ((0, 1), (1234, 2), (4321, 3), (8800, 4)):
        kv[0, table[0][j // ps], 1, j % ps, 2, d] = inf if d % 2 else -inf
    out, lse = cache.attend(0, q.cuda(), causal=False, return_lse=True)
    assert bool((out[0, :, 4:6, 1:4:2] == inf).all()) and bool((out[0, :, 4:6, 2:5:2] == -inf).all())
    assert int((~torch.isfinite(out)).sum()) == T * 2 * 4
    kv[0, table[0][5000 // ps], 0, 5000 % ps, 2, 0] = float("nan")
    nan, lse_nan = cache.attend(0, q.cuda(), causal=False, return_lse=True)
    assert bool(nan[0, :, 4:6].isnan().all()) and bool(lse_nan[0, :, 4:6].isnan().all())
    rest = [h for h in range(8) if h not in (4, 5)]
    assert torch.equal(nan[:, :, rest], out[:, :, rest]) and torch.equal(nan[1], out[1])
