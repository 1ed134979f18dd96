"""Inputs that show a lost low part, for every form of the batched serving
kernels, and what f32's evaluation of them may be off by.

The general bounds (serving_ref.py) count every rounding that a long sum could
make, thousands of times f32's: an evaluation with operands of 11 bits stays
inside them.  Here most keys have no weight and most products are zero, exactly
so in f32, wherever they stand: the sums keep their length and their kernel, but
a dozen roundings are all that there are."""
import numpy as np

import serving_ref as ref

EPS = ref.EPS

# Every form <head class, 32-row groups of a prefix item, of an own item> of the attention kernel by a call that runs it:
# heads, kv, hd, prefix, n, n_q, own, and the tiles that its prefix ranges have at least.
ATTN_FORMS = {
    (64, 1, 1): ((4, 2, 64, 700, 3, 2, 300), 1),
    (64, 2, 1): ((8, 2, 48, 900, 10, 3, 200), 1),
    (64, 2, 2): ((8, 1, 64, 701, 3, 7, 400), 1),
    (64, 4, 1): ((32, 8, 64, 5003, 100, 4, 100), 4),
    (64, 4, 2): ((16, 2, 40, 5003, 60, 6, 150), 4),
    (128, 1, 1): ((32, 4, 128, 1000, 1, 3, 400), 1),
    (128, 2, 1): ((32, 4, 128, 1101, 9, 3, 300), 2),
    (128, 2, 2): ((32, 4, 96, 701, 4, 6, 300), 2),
    (128, 4, 1): ((32, 4, 128, 6001, 64, 4, 150), 6),
    (128, 4, 2): ((32, 4, 128, 9037, 48, 5, 200), 8),
    (256, 1, 1): ((8, 2, 256, 500, 2, 3, 200), 1),
    (256, 2, 1): ((8, 2, 200, 501, 9, 3, 200), 2),
    (256, 2, 2): ((16, 2, 256, 501, 4, 6, 200), 2),
    (256, 4, 1): ((16, 2, 256, 3001, 60, 2, 150), 4),
    (256, 4, 2): ((16, 2, 136, 3001, 40, 5, 100), 4),
}
# Long own ranges, prompts behind a shared prefix, a long verification step.
ATTN_MORE = [(32, 4, 128, 200, 40, 6, 1501), (8, 2, 256, 100, 20, 9, 700), (8, 2, 64, 130, 30, 10, 1100),
             (32, 4, 128, 1000, 1, 260, 260), (8, 2, 64, 300, 2, 333, 500), (8, 2, 256, 200, 1, 150, 190)]
ATTN_LONG = (32, 4, 128, 16384, 64, 5, 640)

# n, rows, cols, rank, adapters: one launch, two for few vectors (by lanes a row of B_e), tiles (by tiles of 16 ranks)
LORA_FORMS = [
    (3, 70, 300, 5, 2), (1, 4096, 2048, 16, 3), (17, 1003, 130, 9, 40), (16, 288, 768, 32, 5), (33, 512, 1000, 64, 7),
    (2, 65, 32801, 8, 2), (3, 70, 16400, 16, 2), (9, 130, 4099, 32, 3), (4, 1001, 3000, 64, 3), (64, 65, 4096, 128, 3),
    (5, 130, 70, 256, 6),
    (6001, 333, 530, 16, 7), (3001, 700, 900, 32, 40), (1500, 700, 900, 64, 9), (1203, 301, 702, 128, 4),
    (700, 331, 521, 256, 5),
]


def _f32(r, *shape):
    """Magnitudes of [1/2, 1) with all their bits, of either sign."""
    return (r.uniform(0.5, 1.0, shape) * r.choice((-1.0, 1.0), shape)).astype(np.float32)


def attn_case(shape, seed=1):
    """Eight prefix rows and up to three of each lane's own have weight (score a sum of three products below 3 in all),
    the others a score of -400."""
    heads, kv, hd, P, n, nq, own = shape
    r = np.random.default_rng([*shape, seed])
    q = _f32(r, n, nq, heads, hd)
    q[..., 0] = 1.0
    q_len = r.integers(1, nq + 1, n).astype(np.int32)
    own_len = r.integers(nq, own + 1, n).astype(np.int32)
    q_len[-1], own_len[-1] = nq, own
    c = {"q": q, "scale": 1.0, "own_len": own_len, "q_len": q_len,
         "kp": np.zeros((P, kv, hd), np.float16), "ko": np.zeros((n, own, kv, hd), np.float16),
         "vp": r.standard_normal((P, kv, hd)).astype(np.float16), "vo": r.standard_normal((n, own, kv, hd)).astype(np.float16)}
    c["kp"][..., 0] = c["ko"][..., 0] = -400.0
    c["live"] = sorted({0, P - 1, min(63, P - 1), min(64, P - 1), min(127, P - 1), P // 2, P * 3 // 4, int(r.integers(P))})
    c["live_own"] = [sorted({0, max(0, int(a) - nq), int(a) - 1}) for a in own_len]

    def enliven(keys, rows):
        for t in rows:
            for h in range(kv):
                keys[t, h, 0] = 0.0
                keys[t, h, 1 + r.choice(hd - 1, 3, replace=False)] = _f32(r, 3)

    enliven(c["kp"], c["live"])
    for i in range(n):
        enliven(c["ko"][i], c["live_own"][i])
    return c


def _f16(x):
    return np.asarray(x, np.float64).astype(np.float16).astype(np.float64)


def attn(c, ragged=True, query=None, weights=None):
    """(out, bound) over the rows that have weight, in 64 bits; `query` and `weights`: what these are rounded by first.

    The bound, with S the largest sum of |q k| of a score and T the rows, in units of 2^-24.  A score: the query in 22
    bits 4 S, six products' sums at a unit of the last place each 12 S, the factor log2 e 2 S, its subtraction from the
    maximum 2 S + 10; the exponential 2; joining key groups, then records, (2 S + 4) each: 24 S + 20 on each weight, once
    in the numerator and once in the sum.  The numerator's weights in 22 bits 4; sums 5 T, rescalings as the maximum moves
    4 T, records 1 T; the quotient 4."""
    n, nq, heads, hd = c["q"].shape
    G = heads // c["kp"].shape[1]
    kp, vp = c["kp"][c["live"]].astype(np.float64), c["vp"][c["live"]].astype(np.float64)
    out, bound = np.full(c["q"].shape, np.nan), np.full(c["q"].shape, np.nan)
    for i in range(n):
        L = int(c["q_len"][i]) if ragged else nq
        length = int(c["own_len"][i])
        rows = c["live_own"][i]
        ko, vo = c["ko"][i, rows].astype(np.float64), c["vo"][i, rows].astype(np.float64)
        k, v = np.concatenate([kp, ko]), np.concatenate([vp, vo])  # [T][kv][hd]
        q = c["q"][i, :L].astype(np.float64).reshape(L, -1, G, hd)
        if query:
            q = query(q)
        s = np.einsum("jhgd,thd->jhgt", q, k)
        S = np.einsum("jhgd,thd->jhgt", np.abs(q), np.abs(k)).max(-1)
        seen = np.arange(L) + length - L + 1
        hidden = np.concatenate([np.zeros((L, len(kp)), bool), np.array(rows)[None, :] >= seen[:, None]], 1)
        s[np.broadcast_to(hidden[:, None, None, :], s.shape)] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        total = p.sum(-1, keepdims=True)
        if weights:
            p = weights(p)
        p /= total
        out[i, :L] = np.einsum("jhgt,thd->jhgd", p, v).reshape(L, heads, hd)
        b = 2 * (24 * S[..., None] + 20) + 4 + 10 * len(k) + 4
        bound[i, :L] = EPS * (b * np.einsum("jhgt,thd->jhgd", p, np.abs(v))).reshape(L, heads, hd)
    return out, bound


def lora_case(shape, seed=1):
    """Every vector has four values that are not zero, and every row of b four ranks."""
    n, rows, cols, rank, adapters = shape
    r = np.random.default_rng([*shape, seed])
    x, b = np.zeros((n, cols), np.float32), np.zeros((adapters, rows, rank), np.float32)
    nx, nb = min(4, cols), min(4, rank)
    at = np.argsort(r.random((n, min(cols, 64))), 1)[:, :nx] * max(1, cols // 64) + cols % max(1, cols // 64)
    at[::3, 0] = cols - 1
    np.put_along_axis(x, at, _f32(r, n, nx), 1)
    bt = np.argsort(r.random((adapters, rows, rank)), 2)[..., :nb]
    np.put_along_axis(b, bt, np.float32(r.choice((-1.0, 1.0, 0.75, -0.625), bt.shape)), 2)
    a = np.float32(r.choice((-1.0, 1.0, 0.75, -0.625, 0.5), (adapters, rank, cols)))
    return {"x": x, "a": a, "b": b, "scale": r.uniform(0.5, 2, adapters).astype(np.float32), "base": _f32(r, n, rows),
            "ids": r.integers(-1, adapters, n).astype(np.int32) if n > 8 else r.integers(0, adapters, n).astype(np.int32)}


def lora(c, vectors=None, inner=None):
    """(out, bound) in 64 bits; `vectors` and `inner`: what x and y = A x are rounded by first.  Both sums have four
    products (a unit of the last place each for the product and the sum: 2 * 4 + 2), then the scale and the addition."""
    x = c["x"].astype(np.float64)
    if vectors:
        x = vectors(x)
    out, bound = c["base"].astype(np.float64), np.zeros(c["base"].shape)
    for e in range(len(c["a"])):
        t = np.nonzero(c["ids"] == e)[0]
        a, b = c["a"][e].astype(np.float64), c["b"][e].astype(np.float64)
        y = x[t] @ a.T
        if inner:
            y = inner(y)
        scale = float(c["scale"][e])
        out[t] += scale * (y @ b.T)
        mag = abs(scale) * (np.abs(x[t]) @ np.abs(a).T) @ np.abs(b).T
        bound[t] = EPS * (24 * mag + 2 * np.abs(out[t]))
    return out, bound


def bf16(x):
    """Rounded to eight significant bits."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.round(m * 256) / 256, e)


f16 = _f16
