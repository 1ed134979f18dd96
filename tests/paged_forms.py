"""Inputs for every form of the attention over pages that show a row that is
missing, doubled or another's, and a lost low part of a query or a weight, and
what f32's evaluation of them may be off by.

The general bound (paged_ref.py) counts every rounding that a long sum could
make: over thousands of rows a tile may be missing inside it, and so may the
low part of an operand.  Here the sums are exact, or a dozen roundings are all
that there are."""
import numpy as np

from serving_ref import EPS


def _many(n, seed, far):
    r = np.random.default_rng(seed)
    lens = r.integers(0, 200, n)
    lens[r.permutation(n)[:n // 8]] = r.integers(600, 2500, n // 8)
    lens[[3, n - 1]] = 0, far
    return [int(x) for x in lens]


# Every form of the kernels by a call that runs it: (whole lanes in one launch, or cut ones with so many waves of the join
# for a query head; head class; whether one block holds a key head's query heads): heads, key heads, head size, page
# size, lens.
FORMS = {
    ("whole", 64, True): (8, 2, 64, 16, [300, 1, 33, 512, 64]),
    ("whole", 64, False): (40, 2, 48, 16, [500, 200, 7]),
    ("whole", 128, True): (32, 4, 128, 16, [512, 100, 31]),
    ("whole", 128, False): (20, 1, 96, 8, [400, 512, 1, 77]),
    ("whole", 256, True): (8, 2, 256, 16, [256, 90, 1]),
    ("whole", 256, False): (18, 1, 200, 16, [255, 130]),
    (2, 64, True): (4, 2, 64, 16, [9000, 300, 40000]),
    (2, 64, False): (36, 2, 48, 24, [20000, 77]),
    (2, 128, True): (4, 1, 128, 16, [33333, 1, 600]),
    (2, 128, False): (20, 1, 128, 7, [12000, 9001]),
    (2, 256, True): (4, 2, 256, 16, [9000, 500]),
    (2, 256, False): (17, 1, 200, 16, [9500]),
    (1, 64, True): (2, 2, 64, 16, _many(150, 1, 20000)),
    (1, 64, False): (34, 2, 40, 24, _many(70, 2, 9000)),
    (1, 128, True): (2, 2, 128, 16, _many(140, 3, 9000)),
    (1, 128, False): (20, 1, 112, 16, _many(130, 4, 12000)),
    (1, 256, True): (2, 2, 256, 5, _many(70, 5, 9000)),
    (1, 256, False): (17, 1, 144, 16, _many(70, 6, 9000)),
}


class Case:
    """Pools of f32 values that f16 and bf16 hold, filled lane by lane; what no lane holds is 1000."""

    def __init__(self, shape, seed):
        self.H, self.KV, self.hd, self.ps, self.lens = shape
        self.r = np.random.default_rng([*shape[:4], len(self.lens), seed])
        n, used = len(self.lens), [-(-x // self.ps) for x in self.lens]
        self.n_pages = sum(used) + 3
        self.table = np.full((n, max(used) + 1), -1, np.int32)
        order, at = self.r.permutation(self.n_pages), 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        self.k, self.v = (np.full((self.n_pages, self.ps, self.KV, self.hd), 1000.0, np.float32) for _ in range(2))
        self.q = np.zeros((n, self.H, self.hd), np.float32)
        self.G = self.H // self.KV

    def rows(self, i):
        t = np.arange(self.lens[i])
        return self.table[i][t // self.ps], t % self.ps

    def first(self, i, window):
        return max(0, self.lens[i] - window) if window else 0


# ---- every row once -------------------------------------------------------------


def coverage_case(shape, by):
    """All scores 0; row t has the value 1 in one column, the next `by` rows in the next one."""
    c = Case(shape, by)
    for i, T in enumerate(c.lens):
        k, v = np.zeros((T, c.KV, c.hd), np.float32), np.zeros((T, c.KV, c.hd), np.float32)
        for h in range(c.KV):
            v[np.arange(T), h, coverage_column(c, i, h, np.arange(T), by)] = 1.0
        c.k[c.rows(i)], c.v[c.rows(i)] = k, v
    return c


def coverage_column(c, i, h, t, by):
    return (t // by + 3 * i + 5 * h) % c.hd


def coverage(c, by, window=0, without=(), twice=()):
    """(out, bound): a column's rows over all rows.  Every sum is of equal powers of two, fewer than 2^24 of them, so
    exact; the reciprocal of the number of rows and the product round.  `without` and `twice`: (lane, row) planted."""
    out = np.zeros(c.q.shape)
    for i, T in enumerate(c.lens):
        t = np.arange(c.first(i, window), T)
        t = np.concatenate([t[~np.isin(t, [x for lane, x in without if lane == i])], [x for lane, x in twice if lane == i]])
        t = t.astype(np.int64)
        for h in range(c.KV):
            n = np.bincount(coverage_column(c, i, h, t, by), minlength=c.hd)
            out[i, h * c.G:(h + 1) * c.G] = n / max(len(t), 1)
    return out, 2 * EPS * out


# ---- one row that outweighs all others, wherever it stands ------------------------


def edge_case(shape):
    """Keys of +-1; a query is 40 times the key of one row, so that every other is 40 times twice their distance below."""
    c = Case(shape, 7)
    for i, T in enumerate(c.lens):
        c.k[c.rows(i)] = c.r.choice(np.float32([-1, 1]), (T, c.KV, c.hd))
        c.v[c.rows(i)] = c.r.integers(-127, 128, (T, c.KV, c.hd))
    return c


def edge_rows(c, turn, window=0):
    """Row [lane][head] that a query is for, -1 where the lane sees none: ends of what is seen, of tiles and units of
    work, more of them every turn."""
    at = np.full((len(c.lens), c.H), -1)
    r = np.random.default_rng([turn, window, c.hd])
    for i, T in enumerate(c.lens):
        first = c.first(i, window)
        if T == first:
            continue
        edges = first + np.arange(0, T - first, 32)
        few = np.concatenate([[first, T - 1] if turn == 0 else [], r.choice(edges, c.H) - r.integers(0, 2, c.H)])
        at[i] = np.clip(few[:c.H], first, T - 1)
    return at


def edges(c, at):
    """The rows' values, exactly; fills in the queries.  Scores are whole numbers, those of other rows 120 lower at least:
    e^-120 of a weight that is exact, which the value's whole number does not feel."""
    want = np.zeros(c.q.shape)
    for i, h in np.argwhere(at >= 0):
        page, row = c.rows(i)
        k = c.k[page, row, h // c.G]
        c.q[i, h] = 40 * k[at[i, h]]
        s = k @ k[at[i, h]]
        assert len(s) == 1 or s[at[i, h]] - np.delete(s, at[i, h]).max() >= 3
        want[i, h] = c.v[page, row, h // c.G][at[i, h]]
    return want


# ---- the query's parts ------------------------------------------------------------


def _live(c, i, h, count):
    """Some rows of a lane: its ends, others anywhere."""
    T = c.lens[i]
    rows = {0, T - 1, *(int(x) for x in np.random.default_rng([i, h, T]).integers(0, T, count))} if T else set()
    return np.array(sorted(rows), np.int64)


def query_case(shape):
    """Up to ten rows of a lane have weight.  Their scores, below 3, are differences of two elements of the query of 32 to
    64: what a query element loses is lost from the score.  Other rows' scores are -400."""
    c = Case(shape, 11)
    c.live = {}
    c.q[:] = c.r.uniform(34, 62, (len(c.lens), c.H, 1)) + c.r.uniform(-1.4, 1.4, c.q.shape)
    c.q[:, :, 0] = 1.0
    for i, T in enumerate(c.lens):
        k, v = np.zeros((T, c.KV, c.hd), np.float32), c.r.integers(-127, 128, (T, c.KV, c.hd)).astype(np.float32)
        k[:, :, 0] = -400.0
        for h in range(c.KV):
            live = c.live[i, h] = _live(c, i, h, 8)
            for t in live:
                a, b = 1 + c.r.choice(c.hd - 1, 2, replace=False)
                k[t, h, [0, a, b]] = 0, 1, -1
        c.k[c.rows(i)], c.v[c.rows(i)] = k, v
    return c


def query(c, kind, rounded=None):
    """(out, bound) over the live rows in 64 bits; `rounded`: what the query is rounded by first.

    The bound, in units of 2^-24.  A score: its sums are of 24 bits from 2^6 down, four roundings at most there (4 * 2^-18
    of the score itself); an f16 cache's query is held in 22 bits, two elements off by 2^-17 each.  The factor log2 e and
    the products 3 S, S < 3; the maximum's subtraction 6, the shift's addition (8.7 + 33 in units of log 2) 29, the
    exponential 2; the running maximum moves up to ten times, then waves and records are joined, 6 + 2 + 1 each for a
    factor: 108.  All of this on each weight, once in the numerator and once in the sum.  The numerator's weights in 22
    bits 2; sums of ten rows, three parts each, twice 30; the quotient 2."""
    out, bound = np.zeros(c.q.shape), np.zeros(c.q.shape)
    score = 4 * 2.0 ** -18 + (2 * 2.0 ** -17 if kind == "f16" else 0.0)
    for i in range(len(c.lens)):
        page, row = c.rows(i)
        for h in range(c.H):
            live = c.live[i, h // c.G]
            if not len(live):
                continue
            k, v = (x[page[live], row[live], h // c.G].astype(np.float64) for x in (c.k, c.v))
            q = c.q[i, h].astype(np.float64)
            s = k @ (rounded(q) if rounded else q)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ v
            bound[i, h] = (2 * score + EPS * (2 * (9 + 6 + 29 + 2 + 108) + 64)) * (p @ np.abs(v))
    return out, bound


# ---- the weights' parts -----------------------------------------------------------


def weight_case(shape):
    """Three rows of one tile of 32 have weight, the values are 1: what comes out is the sum of the weights' parts over the
    sum of the weights, whatever the weights are.  One of them is the largest, with an exact weight."""
    c = Case(shape, 13)
    c.scores = np.zeros((len(c.lens), c.KV, 2))
    for i, T in enumerate(c.lens):
        k = np.zeros((T, c.KV, c.hd), np.float32)
        k[:, :, 0] = -1000.0
        for h in range(c.KV):
            tile = int(c.r.integers(0, max(1, T // 32))) * 32
            live = tile + c.r.permutation(min(32, T - tile))[:3]
            c.scores[i, h] = -c.r.integers(1, 128, 2) / 128.0 if len(live) == 3 else 0
            k[live, h, 0] = [0.0, *c.scores[i, h]][:len(live)]
        c.k[c.rows(i)], c.v[c.rows(i)] = k, 1.0
    return c


WEIGHT_TURNS = 8


def weight_queries(c, turn):
    """Other weights every turn."""
    c.q[:, :, 0] = np.random.default_rng([turn, *c.q.shape]).uniform(0.5, 1.0, c.q.shape[:2])


def weights(c, parts):
    """Each lane's and head's sum of the weights' parts over the sum of the weights, in 64 bits; 0 where there are no rows."""
    s = np.repeat(c.scores, c.G, 1) * c.q[:, :, :1].astype(np.float64)
    w = np.exp(s)
    out = (1 + parts(w).sum(-1)) / (1 + w.sum(-1))
    return np.where(np.array(c.lens)[:, None] >= 3, out, np.array(c.lens)[:, None] > 0)


# Three weights in one tile: an f16 weight in 22 bits (2); three products' sums, of which each may cut off two units of the
# last place (12); the sum of the weights (2); the reciprocal and the product (2).
WEIGHTS_BOUND = 18 * EPS


# ---- operands of fewer parts, for what would show them ---------------------------


def in_parts(bits, parts):
    """x as a sum of numbers of `bits` significant bits each."""

    def rounded(x):
        x = np.asarray(x, np.float64)
        out, left = np.zeros_like(x), x
        for _ in range(parts):
            m, e = np.frexp(left)
            p = np.ldexp(np.round(m * 2.0 ** bits), e - bits)
            out, left = out + p, left - p
        return out

    return rounded


BITS = {"f16": (11, 2), "bf16": (8, 3)}  # of a part, and parts
