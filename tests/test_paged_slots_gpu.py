"""Slots that several requests of an attention call name."""
import pytest
import torch

from tests.test_paged_gpu import TYPES, make
from yapd_b200 import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,T", [(3, 1), (70, 2), (700, 1)])
def test_the_first_request_of_a_slot_stores(dtype, B, T):
    lens = [9, 40, 17, 33]
    cache, q, k, v = make(lens, dtype=TYPES[dtype], T=T, layers=1)
    g = torch.Generator().manual_seed(B)
    slots = torch.randint(0, 4, (B,), generator=g, dtype=torch.int32)
    slots[: min(B, 4)] = torch.tensor([2, 2, 1, 0], dtype=torch.int32)[: min(B, 4)]
    qs, ks, vs = (torch.randn(B, T, 4, 64, generator=g).to(TYPES[dtype]) for _ in range(3))
    want = cache.kv.cpu().clone()
    table = cache.page_table.tolist()
    for s in set(slots.tolist()):
        b = slots.tolist().index(s)
        for i in range(T):
            t = lens[s] - T + i
            want[0, table[s][t // 16], 0, t % 16], want[0, table[s][t // 16], 1, t % 16] = ks[b, i], vs[b, i]
    out = cache.attend(0, qs.cuda(), ks.cuda(), vs.cuda(), slots=slots.cuda())
    assert cache.status() == N.YAPD_STATUS_BAD_SLOT
    assert torch.equal(cache.kv.cpu().view(torch.uint8), want.view(torch.uint8))
    cache.clear_status()
    again = cache.attend(0, qs.cuda(), slots=slots.cuda())      # reading a slot twice is fine
    assert cache.status() == 0 and torch.equal(again, out)


def test_lists_that_begin_anywhere():
    """The list of slots needs no alignment; a slot is found wherever it was named before."""
    lens = [9, 40, 17, 33, 20]
    for start in range(4):
        for at in range(1, 9):
            cache, q, k, v = make(lens, T=1, layers=1)
            names = torch.zeros(start + 9, dtype=torch.int32)
            names[start:] = torch.tensor([0, 1, 2, 3, 9, 9, 9, 9, 9])        # 9: no slot
            names[start + at] = 4
            names[start + 8] = 4
            rows = torch.randn(9, 4, 64).to(torch.bfloat16)
            cache.attend(0, rows.cuda(), rows.cuda(), rows.cuda(), slots=names.cuda()[start:])
            first = at if at < 8 else 8
            page = int(cache.page_table[4, 19 // 16])
            assert torch.equal(cache.kv[0, page, 0, 19 % 16].cpu(), rows[first])
            assert cache.status() == N.YAPD_STATUS_BAD_SLOT
