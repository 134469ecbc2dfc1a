"""KV caches in pages and sampling in numpy: what sequences hold as lists, attention and the sampling rule in f64 (not collected by pytest)."""
import numpy as np

NONE = 0xFFFFFFFF
TYPES = {0: np.float32, 1: np.float16}


class Pool:
    """A pool of pages, its table and its planes [n_planes][n_pages][n_kv][page_rows][hd], which start out as NaN."""

    def __init__(self, n_seqs, max_pages, n_pages, page_rows, n_kv, hd, dtype, n_planes=2):
        self.S, self.max_pages, self.n_pages, self.R, self.n_kv, self.hd, self.dtype = n_seqs, max_pages, n_pages, page_rows, n_kv, hd, dtype
        self.held, self.lens = [[] for _ in range(n_seqs)], [0] * n_seqs
        self.planes = np.full((n_planes, n_pages, n_kv, page_rows, hd), np.nan, TYPES[dtype])

    @property
    def table(self):
        t = np.full((self.S, self.max_pages), NONE, np.uint32)
        for s, pages in enumerate(self.held):
            t[s, :len(pages)] = pages
        return t

    @property
    def refs(self):
        return np.bincount(np.array([p for h in self.held for p in h], int), minlength=self.n_pages).astype(np.uint32)

    def fork(self, parents):
        was = [(list(h), n) for h, n in zip(self.held, self.lens)]
        for s, p in enumerate(parents):
            self.held[s], self.lens[s] = (list(was[p][0]), was[p][1]) if p < self.S else ([], 0)

    def free(self, rows):
        for s, n in enumerate(rows):
            self.held[s] = self.held[s][:-(-n // self.R)]
            self.lens[s] = min(self.lens[s], n)

    def reserve(self, counts):
        """(start, moves, wanting): nothing changes if the last is not 0."""
        refs = self.refs
        free = [p for p in range(self.n_pages) if refs[p] == 0]
        nothing = [NONE] * self.S
        if any(n + c > self.max_pages * self.R for n, c in zip(self.lens, counts)):
            return nothing, [], 0xFFFFFFFF
        writers = {}
        for s, (n, c) in enumerate(zip(self.lens, counts)):
            if c and n % self.R:
                writers.setdefault(self.held[s][n // self.R], []).append(s)
        plan, taken, moves = [], 0, []
        for s, (n, c) in enumerate(zip(self.lens, counts)):
            page = self.held[s][n // self.R] if c and n % self.R else None
            copies = page is not None and not (len(writers[page]) == refs[page] and writers[page][0] == s)
            need = (-(-(n + c) // self.R) + (-n // self.R) + copies) if c else 0
            plan.append((taken, need, copies))
            taken += need
        if taken > len(free):
            return nothing, [], taken - len(free)
        start = list(nothing)
        for s, (at, need, copies) in enumerate(plan):
            if not counts[s]:
                continue
            n = start[s] = self.lens[s]
            new = free[at:at + need]
            if copies:
                moves.append((self.held[s][n // self.R], new[0], n % self.R))
                self.held[s][n // self.R] = new.pop(0)
            self.held[s] += new
            self.lens[s] = n + counts[s]
        return start, moves, 0

    def compact(self):
        used = sorted({p for h in self.held for p in h})
        have = set(used)
        to = [p for p in range(len(used)) if p not in have]
        moves = list(zip([p for p in used if p >= len(used)], to))
        place = dict(moves)
        self.held = [[place.get(p, p) for p in h] for h in self.held]
        return [(a, b, self.R) for a, b in moves], len(used)

    def copy(self, moves):
        for a, b, rows in moves:
            self.planes[:, b, :, :rows] = self.planes[:, a, :, :rows]

    def put(self, s, row, k, v, planes=(0, 1)):
        """[n_kv][hd] of one token at a row of sequence s; dropped where there is no page."""
        if row // self.R >= self.max_pages or row // self.R >= len(self.held[s]):
            return
        page = self.held[s][row // self.R]
        for plane, x in zip(planes, (k, v)):
            with np.errstate(over="ignore"):
                self.planes[plane, page, :, row % self.R] = x.astype(TYPES[self.dtype])

    def rows(self, s, plane):
        """[n_kv][lens[s]][hd] in f64."""
        at = np.array(self.held[s][:-(-self.lens[s] // self.R)], int)
        return self.planes[plane][at].transpose(1, 0, 2, 3).reshape(self.n_kv, -1, self.hd)[:, :self.lens[s]].astype(np.float64)

    def attention(self, q, planes=(0, 1), seen=None):
        """q [S][heads][hd] -> [S][heads][hd] in f64; seen: {sequence: truth value of every row}."""
        out = np.zeros(q.shape)
        group = q.shape[1] // self.n_kv
        for s in range(self.S):
            if self.lens[s] == 0:
                continue
            k, v = self.rows(s, planes[0]), self.rows(s, planes[1])
            there = np.ones(self.lens[s], bool) if seen is None or s not in seen else seen[s]
            if not there.any():
                continue
            for h in range(q.shape[1]):
                x = q[s, h].astype(np.float64) @ k[h // group][there].T / np.sqrt(self.hd)
                e = np.exp(x - x.max())
                out[s, h] = (e / e.sum()) @ v[h // group][there]
        return out


def kept(logits, temperature, top_k, top_p, min_p):
    """(indexes in ascending order, their weights relative to the largest) of what may be taken."""
    x = np.asarray(logits, np.float32).astype(np.float64)
    x[np.isnan(x)] = -np.inf
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    order = np.argsort(-x, kind="stable")
    order = order[:top_k] if 0 < top_k < x.size else order
    order = order[x[order] > -np.inf]
    if order.size == 0:
        return order, np.zeros(0)
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / np.float64(temperature)))
    if top_p < 1:  # (false for NaN)
        w = w[:1 + int(np.searchsorted(np.cumsum(w), max(top_p, 0.0) * w.sum()))][:order.size]
        order = order[:w.size]
    if min_p > 0:
        order, w = order[w >= min(min_p, 1.0)], w[w >= min(min_p, 1.0)]
    by = np.argsort(order)
    return order[by], w[by]


def sample(logits, temperature, top_k, top_p, min_p, u):
    """(token, probability, how far u is from the nearest border of the pick, as a share of the mass)."""
    index, w = kept(logits, temperature, top_k, top_p, min_p)
    if index.size == 0:
        return NONE, 0.0, 1.0
    upto = np.cumsum(w)
    u = 0.0 if np.isnan(u) else min(max(float(u), 0.0), 1.0)
    at = min(int(np.searchsorted(upto, u * upto[-1], side="right")), index.size - 1)
    while w[at] == 0 and at > 0:
        at -= 1
    border = np.abs(np.concatenate([[0.0], upto]) / upto[-1] - u)
    return int(index[at]), w[at] / upto[-1], border[1:-1].min() if index.size > 1 else 1.0
