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
