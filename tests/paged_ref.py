"""The operators around a paged cache in 64 bits, written out lane by lane, and
the error that their f32 evaluation may have (EPS: half an f32 step)."""
import numpy as np

from serving_ref import EPS


def norm_rope(x, pos, freqs, w, eps, interleaved):
    """(y, bound) of x [n][heads][hd]; rows of padding are NaN in both.

    The squares' sum is off by hd/8 + 5 roundings and one a square at most, its mean, root, quotient by one each and half
    of the sum's relative error: 16 + hd / 16 roundings; the two products two.  An angle's turns are rounded to f32 (off
    by pi 2^-25, under two roundings of 1) and the library's sine and cosine are within 4 units in the last place (eight
    half steps); each of the two products and the sum one more.  All relative to |a| + |b| of the pair."""
    x = np.asarray(x, np.float64)
    n, _, hd = x.shape
    y = x.copy()
    if w is not None:
        y = y / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    k = 0 if w is None else 18 + hd / 16
    out, bound = y.copy(), np.abs(y) * k * EPS
    if freqs is not None and len(freqs):
        h = len(freqs)
        a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
        t = np.asarray(pos, np.float64)[:, None] * np.asarray(freqs, np.float64)
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        size = np.abs(y[..., a]) + np.abs(y[..., b])
        bound[..., a] = bound[..., b] = size * (k + 13) * EPS
    pad = np.asarray(pos) < 0
    out[pad], bound[pad] = np.nan, np.nan
    return out, bound


def rounded(x, bound, kind):
    """The bound of values that are rounded once more, to f16 or bf16 (half a step; f16's smallest is 2^-24)."""
    step, least = {"f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}[kind]
    return bound + (np.abs(x) + bound) * step + least


def slots(table, n_pages, page_size, pos, lanes):
    """(page, row) of every token, or None."""
    out = []
    for t, p in enumerate(pos):
        lane = t if lanes is None else int(lanes[t])
        p = int(p)
        ok = p >= 0 and 0 <= lane < len(table) and p // page_size < table.shape[1]
        page = int(table[lane, p // page_size]) if ok else -1
        out.append((page, p % page_size) if 0 <= page < n_pages else None)
    return out


def attn(q, k_pages, v_pages, table, lens, scale, window):
    """(out, bound).  The bound, elementwise: a score is a sum of hd products in f32 (hd roundings, and a query held to 22
    bits: four more) times the scale and log2 e (two), and the exponential's own two; with S = max_t |scale| sum_d |q_d
    k_d| a score is off by (hd + 8) EPS S, its exponential by the same relative amount, numerator and denominator by it
    each.  The weights are held to 22 bits (four), the sums run over T rows (T roundings each, worst case), the joins and
    the division another 32.  All relative to sum_t p_t |v_t|.  Both are held in f16 parts, of which the second has no
    digits below 2^-24: a query element, scaled so that the row's largest is 2^13 at least, and a weight, of which the
    largest is 2^14, are off by up to 2^-25, 2^-38 and 2^-39 of the largest, however small they are themselves."""
    q, k_pages, v_pages = (np.asarray(a, np.float64) for a in (q, k_pages, v_pages))
    n, H, hd = q.shape
    pages, ps, KV = k_pages.shape[:3]
    G = H // KV
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        end = min(max(int(lens[i]), 0), table.shape[1] * ps)
        t = np.arange(max(0, end - window) if window else 0, end)
        page = table[i][t // ps]
        t, page = (a[(page >= 0) & (page < pages)] for a in (t, page))
        if not len(t):
            continue
        k, v = k_pages[page, t % ps], v_pages[page, t % ps]
        for h in range(H):
            kh, vh = k[:, h // G], v[:, h // G]
            s = kh @ q[i, h] * scale
            S = np.max(np.abs(kh) @ np.abs(q[i, h])) * abs(scale)
            small = np.max(np.abs(kh).sum(-1)) * np.abs(q[i, h]).max() * abs(scale) * 2.0 ** -38
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vh
            bound[i, h] = (EPS * (2 * (hd + 8) * S + 4 + 2 * len(t) + 32) + 2 * small) * (p @ np.abs(vh))
            bound[i, h] += 2.0 ** -39 * np.abs(vh).sum(0)
    return out, bound


def logprobs(logits, tokens, top, temperature):
    """(lp, entropy, ids, top_lp) and the bounds of lp, entropy and top_lp.

    With z = (x - max) / T and p its softmax: an exponential is off by |z| (the difference's rounding) and four more
    roundings, the sum of them by the 64 that a thread adds and 32 of the joins; so log S by 2 sum p |z| + 104, a log
    probability by that and its own rounding.  Z / S = sum p z: every term by twice |z| and six, the sums as above."""
    logits = np.asarray(logits, np.float64)
    n, V = logits.shape
    lp, ent = np.full(n, -np.inf), np.zeros(n)
    ids, tops = np.full((n, top), -1, np.int32), np.full((n, top), -np.inf)
    b_lp, b_ent, b_top = np.zeros(n), np.zeros(n), np.zeros((n, top))
    for r, x in enumerate(logits):
        order = np.flatnonzero(~np.isnan(x))
        order = order[np.argsort(-x[order], kind="stable")][:top]
        ids[r, :len(order)] = order
        t = 1.0 if temperature is None else float(temperature[r])
        known = x[~np.isnan(x)]
        m = known.max() if len(known) else -np.inf
        every = np.full(V, -np.inf)
        off = 0.0
        if not t > 0 or 1 / t > 3.4e38 / 1.4427:
            if m > -np.inf:
                every[int(np.flatnonzero(x == m)[0])] = 0.0
        elif np.isnan(x).any() or m == np.inf:
            every[:] = np.nan
            ent[r] = np.nan
        elif m > -np.inf:
            z = np.where(x == -np.inf, -np.inf, (x - m) / t)
            p = np.exp(z)
            S = p.sum()
            p /= S
            every = z - np.log(S)
            live = p > 0
            za = np.abs(z[live]) @ p[live]
            ent[r] = -(p[live] @ every[live])
            off = EPS * (2 * za + 104)
            b_ent[r] = off + EPS * (2 * (z[live] ** 2 @ p[live]) + 110 * za + 2 * abs(ent[r]) + 2)
        with np.errstate(invalid="ignore"):
            own = np.where(np.isfinite(every), off + 2 * EPS * np.abs(every), 0.0)
        if 0 <= tokens[r] < V:
            lp[r], b_lp[r] = every[tokens[r]], own[tokens[r]]
        tops[r, :len(order)], b_top[r, :len(order)] = every[order], own[order]
    return lp, ent, ids, tops, b_lp, b_ent, b_top
