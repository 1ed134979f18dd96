"""The batched serving operators in 64 bits, written out lane by lane, and the
error that their f32 evaluation may have."""
import numpy as np

EPS = 2.0 ** -24  # half an f32 step, relative


def prefix_attn(q, k_pre, v_pre, k_own, v_own, own_len, q_len, scale):
    """(out, bound) of every row of q [n][n_q][H][hd] as float64; rows past q_len are NaN in both.

    The bound, elementwise: a score is a sum of hd products in f32 (hd roundings, and a query held to 22 bits: four
    more) times the scale and log2 e (two), and the exponential's own two; with S = max_t scale * sum_d |q_d k_d| a
    score is off by (hd + 8) EPS S, its exponential by the same relative amount, numerator and denominator by it each.
    The values' weights are held to 22 bits (four), the sums run over T rows (T roundings each, worst case), the merge
    of the parts and the division another 32.  All relative to sum_t p_t |v_t|."""
    n, n_q, H, hd = q.shape
    KV = k_own.shape[2]
    G = H // KV
    q, k_pre, v_pre, k_own, v_own = (np.asarray(a, np.float64) for a in (q, k_pre, v_pre, k_own, v_own))
    out, bound = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    rows = k_own.shape[1]
    for i in range(n):
        L = n_q if q_len is None else min(max(int(q_len[i]), 0), n_q)
        length = min(max(int(own_len[i]), 0), rows)
        for j in range(L):
            seen = max(0, length - L + 1 + j)
            for h in range(H):
                k = np.concatenate([k_pre[:, h // G], k_own[i, :seen, h // G]])
                v = np.concatenate([v_pre[:, h // G], v_own[i, :seen, h // G]])
                if not len(k):
                    out[i, j, h], bound[i, j, h] = 0.0, 0.0
                    continue
                s = k @ q[i, j, h] * scale
                S = np.max(np.abs(k) @ np.abs(q[i, j, h])) * abs(scale)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, j, h] = p @ v
                bound[i, j, h] = EPS * (2 * (hd + 8) * S + 4 + 2 * len(k) + 32) * (p @ np.abs(v))
    return out, bound


def lora(x, a, b, scale, ids, base):
    """(out, bound): cols + rank products and sums, the scale, the widening of nothing, the last addition."""
    x, a, b, scale = (np.asarray(t, np.float64) for t in (x, a, b, scale))
    n, rows = len(x), b.shape[1]
    out = np.zeros((n, rows)) if base is None else np.asarray(base, np.float64).copy()
    bound = np.zeros((n, rows))
    for t in range(n):
        e = int(ids[t])
        if 0 <= e < len(a):
            out[t] += scale[e] * (b[e] @ (a[e] @ x[t]))
            mag = abs(scale[e]) * (np.abs(b[e]) @ (np.abs(a[e]) @ np.abs(x[t])))
            bound[t] = EPS * ((a.shape[2] + a.shape[1] + 4) * mag + 2 * np.abs(out[t]))
    return out, bound


def token_probs(logits, temperature):
    """(p, bound): (x - m) / T in f32 is off by three roundings relative to itself, the exponential by two, the sum by
    one for each value that one thread and then the merge adds (vocab / 256 and 128), the last product by two.  Below
    the smallest normal number a result may be 0."""
    logits = np.asarray(logits, np.float64)
    p, bound = np.zeros_like(logits), np.zeros_like(logits)
    for r, x in enumerate(logits):
        t = 1.0 if temperature is None else float(temperature[r])
        m = x.max()
        if m == -np.inf:
            continue
        if not t > 0:
            p[r, int(np.argmax(x))] = 1.0
            continue
        with np.errstate(over="ignore"):
            z = (x - m) / t
        e = np.exp(z)
        p[r] = e / e.sum()
        bound[r] = p[r] * EPS * (3 * np.abs(np.where(np.isfinite(z), z, 0.0)) + 8 + len(x) / 256 + 128) + 1.2e-38
    return p, bound


def _clean(p):
    p = np.asarray(p, np.float32).astype(np.float64)
    return np.where((p > 0) & (p < np.inf), p, 0.0)


def verify(target, draft, tokens, n_draft, u_accept, u_sample):
    n, k1, vocab = target.shape
    k = k1 - 1
    out, acc = np.full((n, k1), -1, np.int32), np.zeros(n, np.int32)
    for i in range(n):
        nd = k if n_draft is None else min(max(int(n_draft[i]), 0), k)
        r = 0
        while r < nd:
            x = int(tokens[i, r])
            if not 0 <= x < vocab:
                break
            qx = 1.0 if draft is None else _clean(draft[i, r, x])
            if not float(u_accept[i, r]) * float(qx) < float(_clean(target[i, r, x])):
                break
            r += 1
        p = _clean(target[i, r])
        d = p.copy()
        if r < nd:
            if draft is None:
                if 0 <= tokens[i, r] < vocab:
                    d[tokens[i, r]] = 0.0
            else:
                d = np.maximum(p - _clean(draft[i, r]), 0.0)
            if not d.sum() > 0:
                d = p
        out[i, :r] = tokens[i, :r]
        acc[i] = r
        live = np.nonzero(d > 0)[0]
        if len(live):
            c = np.cumsum(d)
            u = float(u_sample[i])
            at = max(u * c[-1], 0.0) if u == u else 0.0
            past = np.nonzero((c > at) & (d > 0))[0]
            out[i, r] = past[0] if len(past) else live[-1]
    return out, acc
