"""The operators of a serving step with drafted tokens restated in float64 numpy
and plain Python, from their definitions in include/foundry_hip.h: the normed
append's norm, tree attention, distributions at a temperature, the verification
of drafted tokens, and the cache's pages."""
import numpy as np

NONE = 0xFFFFFFFF


def norm(x, w, eps):
    """x [.., hd] over its root mean square, times w [hd]; all float64."""
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def visible(width, count, masks=None):
    """[width, width]: whether node i sees node j, rows and nodes past `count` seeing and seen by none."""
    i = np.arange(width)
    if masks is None:
        seen = i <= i[:, None]
    else:
        seen = (masks[:, i // 32] >> (i % 32).astype(np.uint32)) & 1 == 1
    return seen & (i < count) & (i[:, None] < count)


def tree_attend(q, keys, values, table, lengths, counts, masks, scale):
    """q [b, width, heads, hd]; keys, values [pages, kv, page, hd], all float64.
    Returns out, sum p |v| and the largest sum |q||k| * scale of a row."""
    b, width, heads, hd = q.shape
    n_pages, kv, page, _ = keys.shape
    out, weight, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((b, width, heads, 1))
    for s in range(b):
        n, count = int(lengths[s]), min(int(counts[s]), width) if counts is not None else width
        if count == 0 or n + count > table.shape[1] * page:
            continue
        seen = visible(width, count, masks[s] if masks is not None else None)[:, :count]
        at = [(int(table[s, j // page]), j % page) for j in range(n + count)]
        there = np.array([p < n_pages for p, _ in at], bool)
        pages, slots = np.array(at).reshape(-1, 2).T
        pages = np.where(there, pages, 0)
        for h in range(heads):
            k, v = keys[pages, h * kv // heads, slots], values[pages, h * kv // heads, slots]
            for i in range(count):
                use = np.concatenate([np.ones(n, bool), seen[i]]) & there
                if not use.any():
                    continue
                with np.errstate(invalid="ignore"):
                    sc = k[use] @ q[s, i, h] * scale
                    e = np.exp(sc - sc.max())
                    p = e / e.sum()
                    out[s, i, h], weight[s, i, h] = p @ v[use], p @ np.abs(v[use])
                    reach[s, i, h] = (np.abs(k[use]) @ np.abs(q[s, i, h])).max() * scale
    return out, weight, reach


def tree_attend_whole(q, keys, values, table, lengths, counts, masks, scale):
    """tree_attend, all nodes of a head at once, for long contexts."""
    b, width, heads, hd = q.shape
    n_pages, kv, page, _ = keys.shape
    out, weight, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((b, width, heads, 1))
    for s in range(b):
        n, count = int(lengths[s]), min(int(counts[s]), width) if counts is not None else width
        if count == 0 or n + count > table.shape[1] * page:
            continue
        j = np.arange(n + count)
        pages, slots = table[s, j // page].astype(np.int64), j % page
        there = pages < n_pages
        pages = np.where(there, pages, 0)
        seen = visible(width, count, masks[s] if masks is not None else None)[:count, :count]
        seen = np.concatenate([np.ones((count, n), bool), seen], 1) & there
        some = seen.any(1, keepdims=True)
        for h in range(heads):
            k, v = keys[pages, h * kv // heads, slots], values[pages, h * kv // heads, slots]
            sc = np.where(seen, q[s, :count, h] @ k.T * scale, -np.inf)
            e = np.where(seen, np.exp(sc - np.where(some, sc.max(1, keepdims=True), 0)), 0)
            p = e / np.where(some, e.sum(1, keepdims=True), 1)
            bad = ~np.isfinite(v).all(1)  # keys that are added to the rows that see them alone
            out[s, :count, h], weight[s, :count, h] = p[:, ~bad] @ v[~bad], p[:, ~bad] @ np.abs(v[~bad])
            for i in np.nonzero(bad)[0]:
                with np.errstate(invalid="ignore"):
                    out[s, :count, h] += np.where(seen[:, i:i + 1], p[:, i:i + 1] * v[i], 0)
                    weight[s, :count, h] += np.where(seen[:, i:i + 1], p[:, i:i + 1] * np.abs(v[i]), 0)
            reach[s, :count, h, 0] = np.where(seen, np.abs(q[s, :count, h]) @ np.abs(k).T, 0).max(1) * scale
    return out, weight, reach


def probs(z, temperatures=None):
    """softmax(z / t) of each row in float64; z float64 (NaN counts as -inf)."""
    z = np.where(np.isnan(z), -np.inf, z)
    out = np.zeros(z.shape)
    for r in range(z.shape[0]):
        t = float(temperatures[r]) if temperatures is not None else 1.0
        top = z[r].max(initial=-np.inf)
        if top == -np.inf:
            continue
        if not t > 0:
            out[r, int(z[r].argmax())] = 1.0
        elif top == np.inf:
            out[r] = (z[r] == np.inf) / (z[r] == np.inf).sum()
        else:
            e = np.exp((z[r] - top) / min(max(t, 1e-30), 1e30))
            out[r] = e / e.sum()
    return out


def verify(p, q, tokens, parents, counts, u):
    """path, out_tokens, accepted as the definition says it, the weights kept whole.
    p, q (or None) [b, width, n]; tokens, parents (or None) [b, width]."""
    b, width, n = p.shape
    path = np.full((b, width), NONE, np.uint32)
    out = np.full((b, width), NONE, np.uint32)
    accepted = np.zeros(b, np.uint32)
    for s in range(b):
        count = min(int(counts[s]), width) if counts is not None else width
        if count == 0:
            continue
        at, took = 0, [0]
        while True:
            w = np.where(p[s, at] > 0, p[s, at], 0).astype(np.float64)
            total, go = 1.0, None
            for i in range(at + 1, count):
                x = int(tokens[s, i])
                if (int(parents[s, i]) if parents is not None else i - 1) != at or x >= n:
                    continue
                drawn = float(q[s, at, x]) if q is not None else 1.0
                if float(u[s, i]) * drawn * total < w[x]:
                    go = i
                    break
                if q is not None:
                    w = np.maximum(w - total * q[s, at].astype(np.float64), 0)
                    total = w.sum()
                else:
                    total -= w[x]
                    w[x] = 0
            if go is None:
                break
            at = go
            took.append(go)
        if not w.sum() > 0:
            w = np.where(p[s, at] > 0, p[s, at], 0).astype(np.float64)
        sums = w.cumsum()
        past = (sums > float(u[s, 0]) * sums[-1]) & (w > 0)
        word = int(past.argmax()) if past.any() else (int(np.nonzero(w)[0][-1]) if w.any() else NONE)
        accepted[s] = len(took)
        path[s, :len(took)] = took
        out[s, :len(took)] = [int(tokens[s, i]) for i in took[1:]] + [word]
    return path, out, accepted


class Pages:
    """A cache's table, lengths and refs, and [layers, pages, kv, page, hd] pools of plain (ungrouped) keys and values."""

    def __init__(self, table, lengths, refs, k=None, v=None, page=16):
        self.table, self.lengths, self.refs = table.copy(), lengths.copy(), refs.copy()
        self.k, self.v, self.page = (None if k is None else k.copy()), (None if v is None else v.copy()), page
        self.n_pages = len(refs)

    def _take(self, budget):
        if budget[0] == 0:
            return None
        free = np.nonzero(self.refs == 0)[0]
        if len(free) == 0:
            return None
        budget[0] -= 1
        self.refs[free[0]] = 1
        return int(free[0])

    def reserve(self, extra, most=16384):
        missing, budget = np.zeros(len(self.lengths), np.uint32), [most]
        for s, n in enumerate(self.lengths):
            n, x = int(n), int(extra[s])
            if x == 0:
                continue
            first, end, width = n // self.page, -(-(n + x) // self.page), self.table.shape[1]
            missing[s] = max(0, end - max(first, width))
            for e in range(first, min(end, width)):
                if self.table[s, e] >= self.n_pages:
                    got = self._take(budget)
                    missing[s] += got is None
                    self.table[s, e] = NONE if got is None else got
        return missing

    def free(self, seqs):
        for s in seqs:
            if s < len(self.lengths):
                for e in range(self.table.shape[1]):
                    if self.table[s, e] < self.n_pages:
                        self.refs[self.table[s, e]] -= 1
                    self.table[s, e] = NONE
                self.lengths[s] = 0

    def fork(self, src, dst):
        n, (seqs, width) = len(src), self.table.shape
        lost = np.zeros(n, np.uint32)
        for i in range(n):
            if (src[i] >= seqs or dst[i] >= seqs or self.lengths[src[i]] > width * self.page or dst[i] in src
                    or dst[i] in dst[:i]):
                lost[i] = 1
        stand = [i for i in range(n) if not lost[i]]
        for i in stand:
            row = np.full(width, NONE, np.uint32)
            whole = int(self.lengths[src[i]]) // self.page
            row[:whole] = self.table[src[i], :whole]
            row[row >= self.n_pages] = NONE
            for old in self.table[dst[i]]:
                if old < self.n_pages:
                    self.refs[old] -= 1
            for new in row[:whole]:
                if new < self.n_pages:
                    self.refs[new] += 1
            self.table[dst[i]] = row
        budget, undo = [1024], []
        for i in stand:
            length = int(self.lengths[src[i]])
            whole, part = divmod(length, self.page)
            self.lengths[dst[i]] = length
            if part == 0:
                continue
            got = self._take(budget)
            if got is None:
                lost[i] = 1
                undo.append(i)
                continue
            self.table[dst[i], whole] = got
            old = self.table[src[i], whole]
            if old < self.n_pages:
                self.k[:, got, :, :part] = self.k[:, old, :, :part]
                self.v[:, got, :, :part] = self.v[:, old, :, :part]
        self.free([int(dst[i]) for i in undo])
        return lost

    def compact(self, path, accepted):
        for s in range(len(self.lengths)):
            n, row = int(self.lengths[s]), self.table[s]
            for i in range(min(int(accepted[s]), path.shape[1])):
                a, b = n + int(path[s, i]), n + i
                if max(a, b) >= len(row) * self.page or row[a // self.page] >= self.n_pages or row[b // self.page] >= self.n_pages:
                    continue
                for pool in (self.k, self.v):
                    pool[:, row[b // self.page], :, b % self.page] = pool[:, row[a // self.page], :, a % self.page]
        return (self.lengths + np.minimum(accepted, path.shape[1])).astype(np.uint32)
