"""yapd_cache.h: exports, layout, host checks (no GPU needed), and the wrappers' refusals."""
import ctypes as C
import os
import re
import shutil
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "yapd_cache.h")


def test_exports_and_versions():
    from yapd_b200 import _native as N
    from yapd_b200.build import build
    txt = open(HEADER).read()
    declared = set(re.findall(r"^\s*(?:int|size_t)\s+(yapd_\w+)\s*\(", txt, re.M))
    assert declared == set(N.CACHE_EXPORTED)
    lib = C.CDLL(build())
    assert all(hasattr(lib, s) for s in declared)
    assert N.lib().yapd_cache_abi_version() == N.YAPD_CACHE_ABI_VERSION
    for name, value in re.findall(r"#define (YAPD_\w+) (\d+)u?\b", txt):
        assert getattr(N, name) == int(value), name


def test_ctypes_layout_matches_c():
    from yapd_b200 import _native as N
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    structs = {"yapd_cache": N.Cache, "yapd_attend_args": N.AttendArgs, "yapd_pages_args": N.PagesArgs,
               "yapd_logprobs_args": N.LogprobsArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "yapd_cache.h"', "int main(void) {"]
    want = []
    for cname, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        want.append(C.sizeof(py))
        for fname, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {fname}));')
            want.append(getattr(py, fname).offset)
    lines.append("return 0; }")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        open(src, "w").write("\n".join(lines))
        subprocess.run([cc, "-I", os.path.join(ROOT, "include"), "-o", exe, src], check=True)
        got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def good_cache(N):
    c = N.Cache()
    c.layers, c.pages, c.page_size, c.kv_heads, c.head_dim, c.dtype = 2, 10, 16, 4, 64, N.YAPD_DTYPE_BF16
    c.slots, c.max_pages = 3, 8
    c.stride_page = 2 * 16 * 4 * 64
    c.stride_layer = 10 * c.stride_page
    c.kv = c.page_table = c.kv_len = c.refs = c.workspace = 4096      # never dereferenced on the host
    c.workspace_bytes = N.lib().yapd_cache_workspace_size(C.byref(c))
    return c


@pytest.mark.parametrize("field,value,code", [
    ("layers", 0, -2), ("pages", 0, -2), ("page_size", 0, -2), ("page_size", 65537, -2), ("kv_heads", 0, -2),
    ("head_dim", 80, -2), ("slots", 0, -2), ("max_pages", 0, -2), ("max_pages", 2 ** 27, -2), ("dtype", 9, -3),
    ("kv", 0, -1), ("page_table", 0, -1), ("kv_len", 0, -1), ("refs", 0, -1), ("workspace", 0, -1),
    ("kv", 4104, -4), ("stride_page", 2 * 16 * 4 * 64 + 4, -4), ("stride_page", 64, -2), ("stride_layer", 8, -2),
    ("workspace_bytes", 64, -6)])
def test_cache_checks(field, value, code):
    from yapd_b200 import _native as N
    lib = N.lib()
    p, a = N.PagesArgs(), N.AttendArgs()
    p.n, a.B, a.new_tokens, a.heads = 3, 3, 1, 4
    p.cache = a.cache = good_cache(N)
    setattr(p.cache, field, value)
    setattr(a.cache, field, value)
    for name in ("reserve", "fork", "truncate", "trim", "compact", "copy"):
        assert getattr(lib, "yapd_pages_" + name)(C.byref(p), None) == code, name
    assert lib.yapd_attend(C.byref(a), None) == code


def test_call_checks():
    from yapd_b200 import _native as N
    lib = N.lib()
    assert lib.yapd_attend(None, None) == -1 and lib.yapd_pages_reserve(None, None) == -1
    assert lib.yapd_token_logprobs(None, None) == -1
    assert lib.yapd_cache_workspace_size(None) == 0

    def attend(**kw):
        a = N.AttendArgs()
        a.cache = good_cache(N)
        a.B, a.new_tokens, a.heads, a.q, a.out, a.scale = 3, 1, 4, 4096, 4096, 0.125
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.yapd_attend(C.byref(a), None)

    assert attend(B=-1) == -2 and attend(B=4) == -2 and attend(new_tokens=0) == -2 and attend(new_tokens=33) == -2
    assert attend(heads=6) == -2 and attend(heads=0) == -2 and attend(heads=2048) == -2
    assert attend(layer=2) == -8 and attend(layer=-1) == -8 and attend(sinks=-1) == -8
    assert attend(scale=float("nan")) == -8
    assert attend(B=0) == 0
    assert attend(q=None) == -1 and attend(out=None) == -1 and attend(k=4096) == -1 and attend(v=4096) == -1
    assert attend(q=4098) == -4 and attend(q_stride_head=7) == -4 and attend(out_stride_req=4) == -4
    assert attend(k=4096, v=4100) == -4

    def pages(name, **kw):
        p = N.PagesArgs()
        p.cache = good_cache(N)
        p.n = 3
        for k, v in kw.items():
            setattr(p, k, v)
        return getattr(lib, "yapd_pages_" + name)(C.byref(p), None)

    assert pages("reserve", n=4) == -2 and pages("reserve", n=-1) == -2 and pages("reserve", n=0) == 0
    assert pages("fork") == -1 and pages("fork", src=4096) == -1
    assert pages("trim", window=0) == -8 and pages("trim", window=4, sinks=-1) == -8
    assert pages("copy", n=11) == -2 and pages("copy", n=2, src=4096) == -1

    def logprobs(**kw):
        a = N.LogprobsArgs()
        a.R, a.V, a.logits, a.stride_row, a.entropy = 2, 100, 4096, 100, 4096
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.yapd_token_logprobs(C.byref(a), None)

    assert logprobs(R=-1) == -2 and logprobs(V=0) == -2 and logprobs(V=2 ** 20 + 1) == -5
    assert logprobs(top_n=33) == -2 and logprobs(top_n=-1) == -2 and logprobs(top_n=2) == -1
    assert logprobs(logits_dtype=3) == -3 and logprobs(stride_row=99) == -2 and logprobs(logits=None) == -1
    assert logprobs(targets=4096) == -1 and logprobs(logits=4098) == -4 and logprobs(R=0) == 0


def test_wrappers_refuse_cpu_tensors():
    from yapd_b200.logprobs import token_logprobs
    from yapd_b200.paged import PagedCache
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 5))
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache.empty(1, 4, 16, 2, 64, 2, 2, device="cpu")


@pytest.mark.gpu
def test_wrappers_refuse():
    from yapd_b200.logprobs import token_logprobs
    from yapd_b200.paged import PagedCache
    x = torch.zeros(2, 5, device="cuda")
    for bad, kw in ((x.double(), {}), (x[0], {}), (x, dict(top_n=33)), (x, dict(top_n=-1)),
                    (x, dict(targets=torch.zeros(3, dtype=torch.int64, device="cuda"))),
                    (x, dict(targets=torch.zeros(2, device="cuda"))),
                    (x, dict(targets=torch.zeros(2, dtype=torch.int64)))):
        with pytest.raises((TypeError, ValueError)):
            token_logprobs(bad, **kw)
    make = lambda **kw: PagedCache.empty(**{**dict(layers=1, pages=4, page_size=16, kv_heads=2, head_dim=64, slots=2, max_pages=2), **kw})  # noqa: E731
    for kw in (dict(head_dim=48), dict(pages=0), dict(slots=0), dict(dtype=torch.float64), dict(max_pages=0)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            make(**kw)
    c = make()
    with pytest.raises(ValueError):
        PagedCache(c.kv, c.page_table.long(), c.kv_len, c.refs)
    with pytest.raises(ValueError):
        PagedCache(c.kv.transpose(3, 4), c.page_table, c.kv_len, c.refs)
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    slot = torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, kw in (((0, q.float()), {}), ((1, q), {}), ((0, q[:, :1]), {}), ((0, q[..., :32]), {}),
                     ((0, torch.cat([q, q])), {}), ((0, q, q), {}), ((0, q, q, q[:1]), {}),
                     ((0, q, q, q.float()), {}), ((0, q), dict(slots=slot.long())), ((0, q), dict(slots=slot[:1])),
                     ((0, q), dict(sinks=-1)), ((0, q), dict(out=q[:1])), ((0, q.cpu()), {}),
                     ((0, q[:, None].expand(2, 33, 2, 64)), {})):
        with pytest.raises((TypeError, ValueError)):
            c.attend(*args, **kw)
    for call in (lambda: c.reserve(-1), lambda: c.truncate(-2), lambda: c.trim(0), lambda: c.trim(3, -1),
                 lambda: c.reserve(1, slot.long()), lambda: c.fork(slot, slot[:1]),
                 lambda: c.reserve(torch.zeros(3, dtype=torch.int64, device="cuda")),
                 lambda: c.copy_pages(slot, slot.repeat(4))):
        with pytest.raises((TypeError, ValueError)):
            call()
    assert c.status() == 0
