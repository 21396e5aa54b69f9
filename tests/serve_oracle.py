"""Plain 64-bit forms of the operators of include/lg_serve.h, one request, row or key at a time."""
import numpy as np


class Pages:
    """Block table, lengths and stack of free pages, brought up to date the way lg_paged_step describes it."""
    NO_PAGES, TOO_LONG, NO_ROWS, BAD_PAGE = 1, 2, 4, 8

    def __init__(self, table, length, free, n_free, page_size):
        self.table, self.len, self.free = [np.array(a, dtype=np.int64) for a in (table, length, free)]
        self.n_free, self.ps = int(n_free), page_size

    def step(self, new, cap, keep=None):
        ps, columns = self.ps, self.table.shape[1]
        start, pos, slot, req, status, gone = [0], [], [], [], 0, []
        left, out_of_pages, out_of_rows = self.n_free, False, False
        # who is served: pages first, over all requests, then rows among those that have their pages
        plan, taken = [], 0
        for r, n in enumerate(new):
            n = max(0, int(n))
            kept = int(self.len[r]) if keep is None else min(max(0, int(keep[r])), int(self.len[r]))
            have, need = -(-int(self.len[r]) // ps), -(-(kept + n) // ps)
            ok = kept + n <= columns * ps
            status |= 0 if ok else self.TOO_LONG
            if ok and need > have:
                if out_of_pages or taken + need - have > left:
                    ok, out_of_pages = False, True
                    status |= self.NO_PAGES
                else:
                    taken += need - have
            plan.append([ok, kept, n, have, need])
        rows = 0
        for p in plan:
            if p[0] and p[2]:
                if out_of_rows or rows + p[2] > cap:
                    p[0], out_of_rows = False, True
                    status |= self.NO_ROWS
                else:
                    rows += p[2]
        for r, (ok, kept, n, have, need) in enumerate(plan):
            if ok:
                for c in range(have, need):
                    self.n_free -= 1
                    self.table[r, c] = self.free[self.n_free]
                for i in range(kept, kept + n):
                    pos.append(i)
                    slot.append(self.table[r, i // ps] * ps + i % ps)
                    req.append(r)
                gone += [(r, c) for c in range(need, have)]
                self.len[r] = kept + n
            start.append(len(pos))
        for r, c in reversed(gone):
            self.free[self.n_free] = self.table[r, c]
            self.n_free += 1
            self.table[r, c] = -1
        behind = [-1] * (cap - len(pos))
        return start, pos + behind, slot + behind, req + behind, status


def attention(q, k, v, scale, positions, window=0):
    """q [m, heads, dim], k, v [rows, kv_heads, dim] in 64 bits; row t is the query at positions[t]."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    m, heads, dim = q.shape
    group = heads // k.shape[1]
    out = np.zeros((m, heads, dim))
    for t in range(m):
        hi = positions[t] + 1
        lo = max(0, hi - window) if window else 0
        if hi <= lo:
            continue
        for h in range(heads):
            s = k[lo:hi, h // group] @ q[t, h] * scale
            p = np.exp(s - s.max())
            out[t, h] = p @ v[lo:hi, h // group] / p.sum()
    return out


def draw(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row."""
    x = np.asarray(logits, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, 0.0
    first = x[order[0]]
    if not temperature > 0:
        return int(order[0]), 1.0
    if first == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore"):
            w = np.exp((x - first) / np.float64(temperature))
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        run, target, n = 0.0, top_p * w[order].sum(), 0
        cum = np.cumsum(w[order])
        n = 1 + int(np.count_nonzero(cum[:-1] < target))
        order = order[:max(1, n)] if top_p > 0 else order[:1]
    if min_p > 0:
        order = order[:max(1, int(np.count_nonzero(w[order] >= min_p)))]
    kept = np.sort(order)
    cum = np.cumsum(w[kept])
    i = int(np.count_nonzero(cum <= u * cum[-1]))
    if i >= len(kept):
        i = int(np.nonzero(w[kept] > 0)[0][-1])
    return int(kept[i]), float(w[kept[i]] / cum[-1])
