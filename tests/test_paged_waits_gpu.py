"""Calls whose waits expire leave nothing on its way: what runs next on the SM is not disturbed."""
import pytest
import torch

from tests.test_paged_gpu import TYPES, make
from yapd_b200 import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ps", [16, 5])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_copies_land_before_a_cta_ends(dtype, ps):
    """Every CTA holds at most three tiles, so all its copies are issued before a wait of the multiplying
    warps expires; the calls that follow at once take over its shared memory."""
    lens = [37, 64, 200, 1, 5, 129] * 12
    cache, q, k, v = make(lens, dtype=TYPES[dtype], heads=8, kv_heads=4, layers=1, ps=ps)
    q = q.cuda()
    want, want_l = cache.attend(0, q, return_lse=True)
    for _ in range(60):
        cache.attend(0, q, wait_limit_ns=-1)
        out, lse = cache.attend(0, q, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_l)
    assert cache.status() == N.YAPD_STATUS_WAIT_TIMEOUT


@pytest.mark.parametrize("dtype", list(TYPES))
def test_limits_near_the_arrivals(dtype):
    """Limits about as long as the waits take: some expire and some do not, each for a whole warp.
    What was reported as complete is exact, and so is every call that follows."""
    lens = [3000, 37, 700, 0, 64] + [250] * 40
    cache, q, k, v = make(lens, dtype=TYPES[dtype], heads=8, kv_heads=4, layers=1)
    q = q.cuda()
    want, want_l = cache.attend(0, q, return_lse=True)
    for limit in (1, 200, 1000, 2000, 4000, 8000, 20000) * 3:
        cache.clear_status()
        out, lse = cache.attend(0, q, return_lse=True, wait_limit_ns=limit)
        status = cache.status()
        assert status in (0, N.YAPD_STATUS_WAIT_TIMEOUT)
        if status == 0:
            assert torch.equal(out, want) and torch.equal(lse, want_l)
        out, lse = cache.attend(0, q, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_l)
