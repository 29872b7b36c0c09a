"""What of the paged cache can be checked without a GPU."""
import os
import re
import threading
import time

import numpy as np
import pytest
import torch


def test_waits_are_decided_by_whole_warps():
    """No wait of the attention kernel is branched on by a lane alone."""
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yapd_b200", "csrc",
                            "paged_attend.cu")).read()
    assert re.findall(r".*mbar_wait_bounded.*", src) == \
        ["  return __all_sync(~0u, yapd::mbar_wait_bounded(bar, parity, limit_ns));"]


class Recorder:
    """Stands in for the library: each entry notes its arguments, waits, and sees whether they are still the same."""

    def __init__(self):
        self.inside, self.faults, self.calls = 0, [], []

    def __getattr__(self, name):
        def entry(args, stream):
            before = bytes(args)
            self.inside += 1
            time.sleep(2e-4)                    # other threads run
            if self.inside != 1 or bytes(args) != before:
                self.faults.append(name)
            self.inside -= 1
            self.calls.append((name, before))
            return 0
        return entry


@pytest.fixture
def cache(monkeypatch):
    """A cache on CPU tensors whose kernels are not run."""
    from yapd_b200 import _native as N
    from yapd_b200.paged import PagedCache
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    recorder = Recorder()
    recorder.yapd_cache_workspace_size = lambda c: 256
    monkeypatch.setattr(N, "lib", lambda: recorder)

    class Cuda(torch.Tensor):
        is_cuda = True

    kv = torch.zeros(2, 6, 2, 4, 2, 32).as_subclass(Cuda)
    return PagedCache(kv, torch.full((3, 4), -1, dtype=torch.int32), torch.zeros(3, dtype=torch.int64),
                      torch.zeros(6, dtype=torch.int32))


def test_threads_do_not_share_a_call(cache):
    """Each call's arguments are its own, and no two calls' launches mix."""
    from yapd_b200 import _native as N
    made = []

    def attend(i):
        q, k, v = torch.zeros(2, 4, 32), torch.zeros(2, 2, 32), torch.zeros(2, 2, 32)
        slots = torch.zeros(2, dtype=torch.int32)
        out = torch.empty(2, 4, 32)
        for n in range(20):
            cache.attend(i % 2, q, k, v, slots=slots if n % 2 else None, out=out)
            made.append((q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), slots.data_ptr() if n % 2 else None))

    def change(i):
        slots, tokens = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
        for n in range(10):
            cache.reserve(i, slots)
            cache.truncate(tokens, slots)
            cache.fork(slots, slots)
            cache.trim(i + 1, n)
            cache.free()

    threads = [threading.Thread(target=f, args=(i,)) for i in range(3) for f in (attend, change)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not cache._lib.faults
    got = [N.AttendArgs.from_buffer_copy(b) for name, b in cache._lib.calls if name == "yapd_attend"]
    assert sorted(made, key=str) == sorted(((a.q, a.k, a.v, a.out, a.slots) for a in got), key=str) and len(made) == 60
    for name, b in cache._lib.calls:
        if name == "yapd_pages_truncate":
            p = N.PagesArgs.from_buffer_copy(b)
            assert (p.n, p.tokens, p.tokens_each is None) in ((2, 0, False), (3, -1, True))


def test_numbers_that_do_not_fit_are_refused(cache):
    """Nothing is cut off to 64 bits on its way to the library: 2^64 - 1 tokens are not -1, which empties a slot."""
    q = torch.zeros(2, 4, 32)
    for call in (lambda: cache.truncate(2 ** 64 - 1), lambda: cache.truncate(2 ** 64 + 1), lambda: cache.truncate(np.int64(-1)),
                 lambda: cache.reserve(2 ** 63), lambda: cache.reserve(np.int32(-5)), lambda: cache.trim(2 ** 64 + 3),
                 lambda: cache.trim(3, 2 ** 64), lambda: cache.attend(0, q, window=2 ** 63),
                 lambda: cache.attend(0, q, window=5 - 2 ** 64), lambda: cache.attend(0, q, sinks=2 ** 64 + 1)):
        with pytest.raises(ValueError):
            call()
    assert cache._lib.calls == []
    cache.truncate(np.int64(3))
    cache.trim(2 ** 63 - 1, 2 ** 63 - 1)
    cache.attend(0, q, window=2 ** 63 - 1)
    cache.attend(0, q, window=-1)
    assert len(cache._lib.calls) == 4


def test_pages_that_a_copy_could_not_count_are_refused():
    """Half a page of 2^31 vectors of 16 bytes was copied as none."""
    import ctypes as C

    from tests.test_serve_abi import good_cache
    from yapd_b200 import _native as N
    c = good_cache(N)
    c.head_dim, c.kv_heads, c.max_pages = 128, 1024, 2
    for size, dtype, fits in ((32768, N.YAPD_DTYPE_F32, True), (32769, N.YAPD_DTYPE_F32, False),
                              (65536, N.YAPD_DTYPE_F32, False), (65536, N.YAPD_DTYPE_BF16, True)):
        c.page_size, c.dtype = size, dtype
        assert (N.lib().yapd_cache_workspace_size(C.byref(c)) > 0) is fits
