"""64-bit plain implementations of the serving operators, and a host model of the pages."""
import math

import torch

# half a unit in the last place, relative
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend64(keys, values, q, n, *, causal, window, sinks, scale):
    """One request in 64 bits.  keys, values (n, KH, D); q (T, H, D).

    Returns out (T, H, D), lse (T, H), and what the tolerances go by: sum_j p_j |v_j| and the
    largest scale * sum_d |q_d k_d| of a visible token."""
    T, H, D = q.shape
    G = H // keys.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    size = torch.zeros(T, H, D, dtype=torch.float64)
    prod = torch.zeros(T, H, dtype=torch.float64)
    keys, values, q = keys.double(), values.double(), q.double()
    for i in range(T):
        p = n - T + i
        see = [j for j in range(n) if (not causal or j <= p) and (window <= 0 or j > p - window or j < sinks)]
        if not see:
            continue
        k, v = keys[see].repeat_interleave(G, 1), values[see].repeat_interleave(G, 1)
        s = torch.einsum("hd,jhd->hj", q[i], k) * scale
        lse[i] = torch.logsumexp(s, 1)
        w = torch.exp(s - lse[i][:, None])
        w[lse[i] == -math.inf] = 0.0
        out[i] = torch.einsum("hj,jhd->hd", w, v)
        size[i] = torch.einsum("hj,jhd->hd", w, v.abs())
        prod[i] = torch.einsum("hd,jhd->hj", q[i].abs(), k.abs()).amax(1) * scale
    return out, lse, size, prod


def attend_tolerance(dtype, out, size, prod, n, D):
    """Largest errors of out and lse that 32-bit arithmetic explains.

    A score is a sum of D products of inputs, each step rounded to 24 bits, and a product with the
    scale: |ds| <= (D + 4) 2^-24 prod.  The weights err by 2 ds relative (the score's and the
    maximum's), by 2^-21 (1 + 2 prod) from exp (its argument is at most 2 prod away from 0), and
    by 2^-16 where they enter a product as two 16-bit halves.  Sums of n terms lose at most
    (n / 8 + 64) 2^-24 (eight partial sums at least).  The result is rounded once to its type."""
    ds = (D + 4) * 2.0 ** -24 * prod
    rel = 2 * ds + 2.0 ** -21 * (1 + 2 * prod) + (n / 8 + 64) * 2.0 ** -24
    halves = 0.0 if dtype == torch.float32 else 2.0 ** -16
    tol_out = (2 * rel + halves)[..., None] * size + ROUND[dtype] * out.abs() + 2.0 ** -24 * 1e-6
    if dtype == torch.float16:
        tol_out = tol_out + 2.0 ** -25  # the smallest half-precision numbers are 2^-24 apart
    return tol_out, rel + 2.0 ** -22 * (1 + prod)


class Pool:
    """The pages' bookkeeping and contents on the host, one operation at a time."""

    def __init__(self, kv, page_table, kv_len, refs):
        self.kv, self.table = kv.clone(), page_table.tolist()
        self.len, self.refs = kv_len.tolist(), refs.tolist()
        self.ps, self.cols = kv.shape[3], page_table.shape[1]

    def pages_of(self, n):
        return -(-n // self.ps)

    def reserve(self, adds, slots):
        """Pages first, then counts: the list is decided as a whole, on the counts before the call."""
        plan, granted, full = [], [], False
        free = [g for g, r in enumerate(self.refs) if r == 0]
        used = 0
        earlier = {}
        for s, add in zip(slots, adds):
            n = self.len[s]
            if add < 0 or n + add > self.cols * self.ps:
                granted.append(False)
                continue
            first, need, tail = self.pages_of(n), self.pages_of(n + add) - self.pages_of(n), None
            if add > 0 and n % self.ps:
                t = self.table[s][first - 1]
                if t < 0:
                    granted.append(False)
                    continue
                if self.refs[t] > 1:
                    if self.refs[t] - earlier.get(t, 0) > 1:
                        tail, first, need = t, first - 1, need + 1
                    earlier[t] = earlier.get(t, 0) + 1
            full = full or used + need > len(free)
            if full:
                granted.append(False)
                continue
            plan.append((s, add, first, free[used:used + need], tail))
            used += need
            granted.append(True)
        for s, add, first, pages, tail in plan:
            for c, g in enumerate(pages):
                self.table[s][first + c] = g
                self.refs[g] = 1
            if tail is not None:
                k = self.len[s] % self.ps
                self.kv[:, pages[0], :, :k] = self.kv[:, tail, :, :k]
                self.refs[tail] -= 1
            self.len[s] += add
        return granted

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            for c in range(self.pages_of(self.len[a])):
                g = self.table[b][c] = self.table[a][c]
                if g >= 0:
                    self.refs[g] += 1
            self.len[b] = self.len[a]

    def drop(self, s, c):
        g = self.table[s][c]
        if g >= 0:
            self.table[s][c] = -1
            self.refs[g] -= 1

    def truncate(self, takes, slots):
        for s, k in zip(slots, takes):
            keep = self.len[s] - k if 0 <= k <= self.len[s] else 0
            for c in range(self.pages_of(keep), self.pages_of(self.len[s])):
                self.drop(s, c)
            self.len[s] = keep

    def trim(self, window, sinks, slots):
        for s in slots:
            for c in range(self.pages_of(self.len[s])):
                seen = any(j > self.len[s] - window or j < sinks for j in range(c * self.ps, (c + 1) * self.ps))
                if not seen:
                    self.drop(s, c)

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        movers = [g for g in range(live, len(self.refs)) if self.refs[g] > 0]
        holes = [g for g in range(live) if self.refs[g] == 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.kv[:, b] = self.kv[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(g, g) for g in row] for row in self.table]
        return live


def logprobs64(x, targets, top_n):
    """Log softmax of the targets, entropy and alternatives of rows x (R, V), in 64 bits."""
    x = x.double()
    R, V = x.shape
    fine = ~(x.isnan().any(1) | (x == math.inf).any(1) | (x == -math.inf).all(1))
    nan = float("nan")
    # the maximum is taken off first: at 1e38 even 64 bits hold no ln V beside it
    x0 = x - x.amax(1, keepdim=True)
    logp = x0 - x0.exp().sum(1, keepdim=True).log()
    e = logp.exp()
    entropy = torch.where(fine, -torch.special.xlogy(e, e).sum(1), nan)
    spread = torch.where(e > 0, e * x0.abs(), 0.0).sum(1)
    known = (targets >= 0) & (targets < V)
    own = logp.gather(1, targets.clamp(0, V - 1)[:, None])[:, 0]
    own = torch.where(known & fine, own, nan)
    top = torch.full((R, top_n), -math.inf, dtype=torch.float64)
    ids = torch.full((R, top_n), -1, dtype=torch.int64)
    for r in range(R):
        if not fine[r]:
            top[r] = nan
            continue
        order = sorted((v for v in range(V) if x[r, v] > -math.inf), key=lambda v: (-float(x[r, v]), v)) \
            if V <= 4096 else torch.sort(x[r], descending=True, stable=True).indices.tolist()
        order = [v for v in order[:top_n] if x[r, v] > -math.inf]
        ids[r, :len(order)] = torch.tensor(order, dtype=torch.int64)
        top[r, :len(order)] = logp[r, order]
    return own, entropy, top, ids, spread
