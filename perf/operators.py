"""The serving operators' measured cases: attention over a paged key-value cache, the
management of its pages, and token log probabilities.

Each case can be computed in two ways on the same inputs: in plain torch, 32-bit
arithmetic throughout (``own = False``), or through ``yapd_b200.paged`` and
``yapd_b200.logprobs`` (``own = True``).
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}
_DEV = "cuda"


# ----------------------------------------------------------------------------- cases

def _attend(name, **kw):
    case = dict(op="attend", dtype="bf16", batch=1, new=1, heads=16, kv_heads=16, head_dim=64,
                page_size=16, len_min=1, len_max=1, lens=0, causal=True, window=0, sinks=0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _pages(name, **kw):
    case = dict(op="draft", dtype="bf16", layers=24, requests=1, beams=1, kv_heads=16, head_dim=64,
                page_size=16, len_min=1, len_max=1, lens=0, tokens=1, window=0, sinks=0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _logprobs(name, **kw):
    case = dict(op="logprobs", dtype="f32", rows=1, vocab=6563, top_n=0, pad=0, masked=0.0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one autoregressive request mid-utterance: the latency of a single call
        _attend("attend_one", batch=1, len_min=417, len_max=417),
        # a full autoregressive tick: 256 requests at ragged lengths, every head with its own keys
        _attend("attend_tick", batch=256, len_min=20, len_max=1250, lens=1),
        # a block-diffusion step: 16 positions that see one another, conditional and unconditional rows
        _attend("attend_block", batch=128, new=16, causal=False, len_min=60, len_max=1100, lens=2),
        # a few very long contexts with shared key heads: the split over the length carries the call
        _attend("attend_long", dtype="f16", batch=4, heads=32, kv_heads=8, head_dim=128, page_size=64,
                len_min=60001, len_max=131072, lens=3),
        # long-running streams: the prompt stays visible, the rest slides
        _attend("attend_window", batch=48, heads=16, kv_heads=4, head_dim=128, len_min=3000, len_max=30000,
                lens=4, window=2000, sinks=150),
        # a 32-bit model with odd pages and a short causal draft
        _attend("attend_f32", dtype="f32", batch=24, new=5, heads=8, kv_heads=4, page_size=5, len_min=5,
                len_max=901, lens=5),
        # a refused draft: five tokens reserved and given back for every request of a tick (bookkeeping
        # alone, whatever the layers: one stands for all)
        _pages("pages_draft", op="draft", layers=1, requests=256, len_min=20, len_max=1250, lens=6, tokens=5),
        # candidates of 64 requests replaced: the losers freed, the winners forked, their tail pages unshared
        _pages("pages_fork", op="fork", requests=64, beams=4, len_min=33, len_max=1200, lens=7, tokens=1),
        # a long-running pool: what left the windows is freed and the pool packed to its low end
        _pages("pages_pack", op="pack", requests=20, len_min=400, len_max=2600, lens=8, window=500, sinks=64),
        # the sampled token of one request, with alternatives
        _logprobs("logprobs_one", rows=1, vocab=6563, top_n=5),
        # every position of a block-diffusion batch (odd vocabulary: rows are not vector-aligned)
        _logprobs("logprobs_block", dtype="bf16", rows=8192, vocab=8194, top_n=8),
        # scoring with a large text vocabulary under a grammar mask
        _logprobs("logprobs_text", dtype="bf16", rows=384, vocab=128256, top_n=20, masked=0.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "pages", "logprobs", "logprobs"])
    if kind == "attend":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        dim = rng.choice([32, 64, 64, 96, 128])
        kvh = rng.choice([1, 2, 3, 4, 8, 16])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        new = rng.choice([1, 1, 1, rng.randint(2, 32), 16])
        longest = _log(rng, 1, 131072)
        room = 5e8 / (2 * kvh * dim * 4) / longest      # the plain form's 32-bit gather stays below 0.5 GB a side
        room = min(room, 1e9 / (4 * kvh * group * new) / longest)
        batch = max(1, min(_log(rng, 1, 300), int(room)))
        longest = max(new, min(longest, int(max(room, 1.0) / max(1, batch) * longest) + 1))
        windowed = rng.random() < 0.4
        return _attend(None, dtype=dtype, batch=batch, new=new, heads=kvh * group, kv_heads=kvh, head_dim=dim,
                       page_size=rng.choice([1, 5, 8, 16, 16, 32, 64, 100]),
                       len_min=rng.choice([new, max(new, longest // 2)]), len_max=longest, lens=rng.randint(1, 10 ** 6),
                       causal=rng.random() < 0.6, window=_log(rng, 1, longest + 8) if windowed else 0,
                       sinks=_log(rng, 1, 300) - 1 if windowed else 0)
    if kind == "pages":
        op = rng.choice(["draft", "fork", "pack"])
        longest = _log(rng, 16, 3000)
        layers = rng.randint(1, 30)
        kvh, dim = rng.choice([2, 4, 8, 16]), rng.choice([32, 64, 96, 128])
        dtype = rng.choice(["bf16", "f16", "f32"])
        token = layers * 2 * kvh * dim * _SIZES[dtype]
        beams = rng.randint(2, 8) if op == "fork" else 1
        requests = max(1, min(_log(rng, 1, 512), int(3e9 / token / longest / (2 if op == "fork" else 1))))
        return _pages(None, op=op, dtype=dtype, layers=layers, requests=requests, beams=beams, kv_heads=kvh,
                      head_dim=dim, page_size=rng.choice([1, 7, 16, 16, 32, 64]), len_min=max(1, longest // 20),
                      len_max=longest, lens=rng.randint(1, 10 ** 6), tokens=rng.randint(1, 40),
                      window=_log(rng, 8, longest) if op == "pack" else 0,
                      sinks=rng.randint(0, 100) if op == "pack" else 0)
    vocab = _log(rng, 2, 262144)
    dtype = rng.choice(["bf16", "f16", "f32"])
    return _logprobs(None, dtype=dtype, rows=max(1, min(_log(rng, 1, 16384), int(1.2e8 / vocab))), vocab=vocab,
                     top_n=rng.choice([0, 1, 5, 20, 32]), pad=rng.choice([0, 0, 1, 6]),
                     masked=rng.choice([0.0, 0.0, 0.3, 0.9]))


def _lengths(case, n):
    r = random.Random(case["lens"])
    return [r.randint(case["len_min"], case["len_max"]) for _ in range(n)]


# ----------------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed))
    return g


def _tables(lens, ps, columns, pages, g):
    """Page tables of requests with `lens` tokens, on pages in random order; and the pages' reference counts."""
    held = [-(-n // ps) for n in lens]
    order = torch.randperm(pages, generator=g, device=_DEV).to(torch.int32)
    table = torch.full((len(lens), columns), -1, dtype=torch.int32, device=_DEV)
    counts = torch.tensor(held, device=_DEV)
    col = torch.arange(columns, device=_DEV)
    inside = col[None, :] < counts[:, None]
    table[inside] = order[: sum(held)]
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEV)
    refs[order[: sum(held)].long()] = 1
    return table, refs


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "logprobs":
        return _prepare_logprobs(case, g)
    if case["op"] == "attend":
        return _prepare_attend(case, g)
    return _prepare_pages(case, g)


def _handle(state):
    """The cache's handle, which a program keeps for as long as the pool lives."""
    if own:
        from yapd_b200.paged import PagedCache
        state["cache"] = PagedCache(state["kv"], state["page_table"], state["kv_len"], state["refs"])
    return state


def _prepare_attend(case, g):
    dt, ps, B, new = _TYPES[case["dtype"]], case["page_size"], case["batch"], case["new"]
    D, H, KH = case["head_dim"], case["heads"], case["kv_heads"]
    lens = _lengths(case, B)
    columns = max(-(-n // ps) for n in lens) + 1
    pages = sum(-(-n // ps) for n in lens) + 3
    table, refs = _tables(lens, ps, columns, pages, g)
    kv = torch.empty(1, pages, 2, ps, KH, D, dtype=dt, device=_DEV).normal_(generator=g)
    # queries a little larger than unit variance: the softmax has its peaks, as trained heads have
    q = (torch.randn(B, new, H, D, generator=g, device=_DEV) * 1.5).to(dt)
    k = torch.randn(B, new, KH, D, generator=g, device=_DEV).to(dt)
    v = torch.randn(B, new, KH, D, generator=g, device=_DEV).to(dt)
    kv_len = torch.tensor(lens, dtype=torch.int64, device=_DEV)
    return _handle(dict(case=case, kv=kv, page_table=table, kv_len=kv_len, refs=refs, q=q, k=k, v=v))


def _prepare_pages(case, g):
    dt, ps, n, op = _TYPES[case["dtype"]], case["page_size"], case["requests"], case["op"]
    lens = _lengths(case, n)
    columns = -(-(case["len_max"] + case["tokens"]) // ps) + 1
    held = sum(-(-x // ps) for x in lens)
    spare = {"draft": n * (case["tokens"] // ps + 2), "pack": held // 3 + 5,
             "fork": n * (case["beams"] - 1) * (case["tokens"] // ps + 2)}[op] + 7
    table, refs = _tables(lens, ps, columns, held + spare, g)
    kv = torch.empty(case["layers"], held + spare, 2, ps, case["kv_heads"], case["head_dim"], dtype=dt,
                     device=_DEV).normal_(generator=g)
    kv_len = torch.tensor(lens, dtype=torch.int64, device=_DEV)
    state = dict(case=case, kv=kv)
    if op == "fork":
        # slot r * beams holds request r; the other slots of its beam hold candidates that lose
        beams = case["beams"]
        wide = torch.full((n * beams, columns), -1, dtype=torch.int32, device=_DEV)
        wide[::beams] = table
        lens_wide = torch.zeros(n * beams, dtype=torch.int64, device=_DEV)
        lens_wide[::beams] = kv_len
        slot = torch.arange(n * beams, device=_DEV, dtype=torch.int32)
        state["dst"] = slot[slot % beams != 0].contiguous()
        state["src"] = (state["dst"] // beams * beams).contiguous()
        table, kv_len = wide, lens_wide
    if op == "pack":
        # the bookkeeping before the pass: every pass packs the same pool again
        state["before"] = (table.clone(), kv_len.clone(), refs.clone())
    state.update(page_table=table, kv_len=kv_len, refs=refs)
    return _handle(state)


def _prepare_logprobs(case, g):
    R, V, dt = case["rows"], case["vocab"], _TYPES[case["dtype"]]
    x = torch.empty(R, V + case["pad"], dtype=dt, device=_DEV).normal_(0.0, 2.0, generator=g)[:, :V]
    # a few tokens stand out of the noise in every row, as a language model's logits do
    k = min(12, V)
    at = (torch.randint(0, V, (R, 1), generator=g, device=_DEV) + torch.arange(k, device=_DEV) * (V // k)) % V
    x.scatter_(1, at, (torch.randn(R, k, generator=g, device=_DEV) * 3 + 9).to(dt))
    if case["masked"]:
        x.masked_fill_(torch.rand(R, V, generator=g, device=_DEV) < case["masked"], float("-inf"))
        x[:, V - 1] = 1.0  # the end token is never masked
    targets = at[:, 0].clone()
    targets[5::17] = -1   # positions without a token
    return dict(case=case, logits=x, targets=targets)


# ----------------------------------------------------------------------------- passes

def run(state):
    op = state["case"]["op"]
    if op == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    if op == "logprobs":
        return _own_logprobs(state) if own else _plain_logprobs(state)
    return _own_pages(state) if own else _plain_pages(state)


def _own_attend(state):
    c = state["case"]
    out, lse = state["cache"].attend(0, state["q"], state["k"], state["v"], causal=c["causal"],
                                     window=c["window"], sinks=c["sinks"], return_lse=True)
    return {"out": out, "lse": lse, "kv": state["kv"]}


def _own_pages(state):
    c, cache = state["case"], state["cache"]
    got = {}
    if c["op"] == "draft":
        got["granted"] = cache.reserve(c["tokens"])
        got["drafted"] = state["page_table"].clone()
        cache.truncate(c["tokens"])
    elif c["op"] == "fork":
        cache.free(state["dst"])
        cache.fork(state["src"], state["dst"])
        got["granted"] = cache.reserve(c["tokens"], state["dst"])
    else:
        _restore(state)
        cache.trim(c["window"], c["sinks"])
        got["live"] = cache.compact()
    return {**got, "page_table": state["page_table"], "kv_len": state["kv_len"], "refs": state["refs"],
            "kv": state["kv"]}


def _own_logprobs(state):
    from yapd_b200.logprobs import token_logprobs
    r = token_logprobs(state["logits"], state["targets"], top_n=state["case"]["top_n"])
    got = {"logprob": r.logprob, "entropy": r.entropy}
    if state["case"]["top_n"]:
        got.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
    return got


def _restore(state):
    for name, saved in zip(("page_table", "kv_len", "refs"), state["before"]):
        state[name].copy_(saved)


def _plain_attend(state):
    c, kv, table, n = state["case"], state["kv"], state["page_table"], state["kv_len"]
    q, new, ps = state["q"], c["new"], c["page_size"]
    B, _, H, D = q.shape
    KH = c["kv_heads"]
    # the new tokens' rows go to their places in the pages
    at = n[:, None] - new + torch.arange(new, device=q.device)
    page = table.gather(1, at // ps).long()
    kv[0, page, 0, at % ps] = state["k"]
    kv[0, page, 1, at % ps] = state["v"]
    # the pages of each request side by side, in 32 bits
    held = kv[0, table.clamp_min(0).long()].float()                # (B, columns, 2, ps, KH, D)
    key = held[:, :, 0].reshape(B, -1, KH, D).permute(0, 2, 3, 1)  # (B, KH, D, N)
    value = held[:, :, 1].reshape(B, -1, KH, D).permute(0, 2, 1, 3)
    N = key.shape[-1]
    rows = q.float().reshape(B, new, KH, H // KH, D).permute(0, 2, 1, 3, 4).reshape(B, KH, -1, D)
    s = (rows @ key) / math.sqrt(D)
    j = torch.arange(N, device=q.device)
    p = at[:, :, None]
    seen = (j < n[:, None, None]).expand(B, new, N)
    if c["causal"]:
        seen = seen & (j <= p)
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["sinks"]))
    seen = seen[:, None, :, None, :].expand(B, KH, new, H // KH, N).reshape(B, KH, -1, N)
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = (s - m).exp()
    z = e.sum(-1, keepdim=True)
    value = value.masked_fill((j >= n[:, None])[:, None, :, None], 0.0)
    o = (e @ value) / z
    o = o.reshape(B, KH, new, H // KH, D).permute(0, 2, 1, 3, 4).reshape(B, new, H, D).to(q.dtype)
    lse = (m + z.log()).reshape(B, KH, new, H // KH).permute(0, 2, 1, 3).reshape(B, new, H)
    return {"out": o, "lse": lse, "kv": kv}


def _plain_count(refs, pages, step):
    """Adds `step` to the count of each page of `pages` (-1: none)."""
    flat = pages.reshape(-1).long()
    refs.index_add_(0, flat.clamp_min(0), (flat >= 0).to(torch.int32) * step)


def _plain_reserve(state, tokens, slots):
    """`tokens` more for each of `slots`, in order, on the lowest free pages; a tail page that is shared is copied."""
    kv, table, refs, ps = state["kv"], state["page_table"], state["refs"], state["case"]["page_size"]
    before = state["kv_len"][slots]
    rows = table[slots]
    have = (before + ps - 1) // ps
    need = (before + tokens + ps - 1) // ps - have
    last = (have - 1).clamp_min(0)
    tail = rows.gather(1, last[:, None])[:, 0].long()
    part = before % ps
    same = (tail[:, None] == tail[None, :]) & (part != 0)[None, :]
    earlier = same.tril(-1).sum(1)
    copied = (part != 0) & (refs[tail.clamp_min(0)] - earlier > 1)
    count = need + copied
    upto = count.cumsum(0)
    granted = upto <= (refs == 0).sum()
    free = torch.argsort((refs != 0).to(torch.int32), stable=True)      # free pages first, lowest first
    col = torch.arange(rows.shape[1], device=rows.device)
    first = torch.where(copied, last, have)
    taken = granted[:, None] & (col >= first[:, None]) & (col < (first + count)[:, None])
    source = (upto - count)[:, None] + col - first[:, None]
    fresh = free[source.clamp(0, free.numel() - 1)].to(torch.int32)
    rows = torch.where(taken, fresh, rows)
    moved = copied & granted
    fresh_tail = rows.gather(1, last[:, None])[:, 0].long()
    a, b = tail[moved], fresh_tail[moved]
    held = torch.arange(ps, device=rows.device) < part[moved][:, None]
    held = held[None, :, None, :, None, None]
    kv[:, b] = torch.where(held, kv[:, a], kv[:, b])
    _plain_count(refs, torch.where(moved, tail, -1), -1)
    _plain_count(refs, torch.where(taken, rows, -1), 1)
    table[slots] = rows
    state["kv_len"][slots] = before + tokens * granted
    return granted


def _plain_drop(state, slots, keep):
    """The pages of `slots` past their first `keep` tokens go."""
    table, ps = state["page_table"], state["case"]["page_size"]
    rows = table[slots]
    gone = torch.arange(rows.shape[1], device=rows.device) >= ((keep + ps - 1) // ps)[:, None]
    _plain_count(state["refs"], torch.where(gone, rows, -1), -1)
    table[slots] = torch.where(gone, -1, rows)
    state["kv_len"][slots] = keep


def _plain_trim(state, window, sinks):
    """Pages that lie between the first `sinks` tokens and what the next token's window reaches go."""
    table, n, ps = state["page_table"], state["kv_len"], state["case"]["page_size"]
    start = torch.arange(table.shape[1], device=table.device) * ps
    reach = (n + 1 - window)[:, None]                    # the next token, at n, sees j > n - window
    gone = (start >= sinks) & (start + ps <= reach) & (table >= 0)
    _plain_count(state["refs"], torch.where(gone, table, -1), -1)
    table.copy_(torch.where(gone, -1, table))


def _plain_pack(state):
    """Live pages past the first `live` pages move, in order, into the free ones among those."""
    kv, table, refs = state["kv"], state["page_table"], state["refs"]
    used = refs > 0
    live = used.sum()
    low = torch.arange(refs.numel(), device=refs.device) < live
    a, b = (used & ~low).nonzero()[:, 0], (~used & low).nonzero()[:, 0]
    kv[:, b] = kv[:, a]
    refs[b] = refs[a]
    refs[a] = 0
    to = torch.arange(refs.numel(), device=refs.device, dtype=torch.int32)
    to[a] = b.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()], -1))
    return live.to(torch.int32).reshape(1)


def _plain_pages(state):
    c = state["case"]
    got = {}
    if c["op"] == "draft":
        slots = torch.arange(c["requests"], device=_DEV)
        got["granted"] = _plain_reserve(state, c["tokens"], slots)
        got["drafted"] = state["page_table"].clone()
        _plain_drop(state, slots, state["kv_len"] - c["tokens"])
    elif c["op"] == "fork":
        src, dst = state["src"].long(), state["dst"].long()
        _plain_drop(state, dst, torch.zeros_like(dst))
        state["page_table"][dst] = state["page_table"][src]
        state["kv_len"][dst] = state["kv_len"][src]
        _plain_count(state["refs"], state["page_table"][dst], 1)
        got["granted"] = _plain_reserve(state, c["tokens"], dst)
    else:
        _restore(state)
        _plain_trim(state, c["window"], c["sinks"])
        got["live"] = _plain_pack(state)
    return {**got, "page_table": state["page_table"], "kv_len": state["kv_len"], "refs": state["refs"],
            "kv": state["kv"]}


def _plain_logprobs(state):
    x, t, n = state["logits"].float(), state["targets"], state["case"]["top_n"]
    V = x.shape[1]
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    logp = x - m - z.log()
    entropy = -torch.where(e > 0, e / z * logp, torch.zeros_like(logp)).sum(-1)
    own_token = logp.gather(1, t.clamp_min(0)[:, None])[:, 0]
    got = {"logprob": torch.where(t >= 0, own_token, float("nan")), "entropy": entropy}
    if n:
        top, ids = x.sort(dim=-1, descending=True, stable=True)
        top, ids = top[:, :n], ids[:, :n].to(torch.int32)
        ids = torch.where(top > float("-inf"), ids, -1)
        top = top - m - z.log()
        more = n - top.shape[1]                          # a vocabulary smaller than n
        got["top_logprobs"] = torch.nn.functional.pad(top, (0, more), value=float("-inf")) if more > 0 else top
        got["top_ids"] = torch.nn.functional.pad(ids, (0, more), value=-1) if more > 0 else ids
    return got


# ----------------------------------------------------------------------------- work

def _visible(case, n):
    """Keys of a request of `n` tokens that at least one of its new tokens sees, and (new token, key) pairs."""
    new, window, sinks = case["new"], case["window"], case["sinks"]
    pairs = 0
    for i in range(new):
        p = n - new + i
        end = p + 1 if case["causal"] else n
        low = max(0, p - window + 1) if window else 0
        pairs += end - low + min(sinks, low) if window else end
    low = max(0, n - new - window + 1) if window else 0
    return n - low + min(sinks, low), pairs


def work(case):
    s = _SIZES[case["dtype"]]
    if case["op"] == "attend":
        KH, H, D, new, ps = case["kv_heads"], case["heads"], case["head_dim"], case["new"], case["page_size"]
        seen = [_visible(case, n) for n in _lengths(case, case["batch"])]
        keys, pairs = sum(k for k, _ in seen), sum(p for _, p in seen)
        rows = case["batch"] * new
        # the new rows are read from the call's k and v and written to the pages
        moved = 2 * KH * D * s * (keys + rows) + 2 * rows * H * D * s + 4 * rows * H
        return {"bytes": moved + sum(4 * -(-k // ps) for k, _ in seen) + 8 * case["batch"], "flops": 4 * D * H * pairs}
    if case["op"] == "logprobs":
        R, V, n = case["rows"], case["vocab"], case["top_n"]
        return {"bytes": R * (V * s + 8 + 8 + 8 * n), "flops": 6 * R * V}
    ps, n = case["page_size"], case["requests"]
    lens = _lengths(case, n)
    token = case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * s
    held = sum(-(-x // ps) for x in lens)
    if case["op"] == "draft":
        return {"bytes": 4 * (held + 2 * n) + 40 * n, "flops": 0}
    if case["op"] == "fork":
        forks = case["beams"] - 1
        copied = sum(x % ps for x in lens) * forks
        return {"bytes": 2 * token * copied + 12 * held * forks + 40 * n * forks, "flops": 0}
    kept = sum(sum(1 for a in range(0, x, ps) if not (a >= case["sinks"] and a + ps <= x + 1 - case["window"]))
               for x in lens)
    pages = held + held // 3 + 12
    moved = kept * (pages - kept) // pages               # expected: live pages spread evenly over the pool
    return {"bytes": 2 * token * ps * moved + 12 * held + 8 * pages, "flops": 0}


# ----------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    if case["op"] == "logprobs":
        return _exact_logprobs(case, prepare(case, seed))
    if case["op"] == "attend":
        return _exact_attend(case, prepare(case, seed))
    return None  # copies and whole numbers only


def _exact_attend(case, state):
    """One request at a time, its tokens looked up one by one."""
    ps, new, D = case["page_size"], case["new"], case["head_dim"]
    group = case["heads"] // case["kv_heads"]
    outs, lses = [], []
    for b, n in enumerate(_lengths(case, case["batch"])):
        j = torch.arange(n, device=_DEV)
        page = state["page_table"][b].long()[torch.div(j, ps, rounding_mode="floor")]
        key = state["kv"][0][page, 0, j % ps].double()
        val = state["kv"][0][page, 1, j % ps].double()
        key[n - new:], val[n - new:] = state["k"][b].double(), state["v"][b].double()
        key, val = key.repeat_interleave(group, 1), val.repeat_interleave(group, 1)   # (n, H, D)
        score = torch.einsum("ihd,jhd->hij", state["q"][b].double(), key) * D ** -0.5
        place = torch.arange(n - new, n, device=_DEV)[:, None]
        hidden = (j[None] > place) if case["causal"] else torch.zeros(new, n, dtype=torch.bool, device=_DEV)
        if case["window"]:
            hidden = hidden | ((place - j[None] >= case["window"]) & (j[None] >= case["sinks"]))
        score[hidden.expand_as(score)] = -math.inf
        total = torch.logsumexp(score, -1)
        outs.append(torch.einsum("hij,jhd->ihd", torch.exp(score - total[..., None]), val))
        lses.append(total.transpose(0, 1))
    return {"out": torch.stack(outs), "lse": torch.stack(lses), "kv": None}


def _exact_logprobs(case, state):
    x, t, n = state["logits"].double(), state["targets"], case["top_n"]
    total = torch.logsumexp(x, 1)
    logp = x - total[:, None]
    entropy = -torch.special.xlogy(logp.exp(), logp.exp()).sum(1)
    one = logp[torch.arange(len(t), device=t.device), t.clamp_min(0)]
    one[t < 0] = math.nan
    got = {"logprob": one, "entropy": entropy}
    if n:
        best = torch.topk(logp, min(n, logp.shape[1]), 1).values
        full = torch.full((len(t), n), -math.inf, dtype=torch.float64, device=t.device)
        full[:, : best.shape[1]] = best
        got.update(top_logprobs=full, top_ids=None)
    return got
