"""The operators of serving from a paged key-value cache as measurable cases:
norms and rotation of queries and keys, appending them to the cache's pages,
attention of each request's new token over its pages, and the log
probabilities of the tokens that come out.

`run` computes each in its plain form (elementary torch operations in 32 bits,
64 for the angles of far positions), or, where `own` is set, through
loom_amd.serving.  Sizes are those of the repository's own configurations (the
Qwen3-30B-A3B and stories15M shapes: heads, head size, vocabularies, the
4096-token context, 32 and 64 lanes) or generic ragged ones.
"""
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request after a short prompt, its next token: the latency of a call
        {"name": "attn_token", "kind": "attn", "heads": 32, "kv": 4, "hd": 128, "n": 1, "rows": 256, "page": 16,
         "type": "f16", "window": 0},
        # the small dense model's heads (no sharing of key heads), odd sizes, pages of an odd length
        {"name": "attn_ragged", "kind": "attn", "heads": 6, "kv": 6, "hd": 48, "n": 5, "rows": 1003, "page": 24,
         "type": "bf16", "window": 0},
        # ordinary batched decode: 32 requests with up to 4096 tokens
        {"name": "attn_lanes", "kind": "attn", "heads": 32, "kv": 4, "hd": 128, "n": 32, "rows": 4096, "page": 16,
         "type": "f16", "window": 0},
        # a few requests over long documents, bf16, large pages
        {"name": "attn_long", "kind": "attn", "heads": 32, "kv": 4, "hd": 128, "n": 8, "rows": 65536, "page": 64,
         "type": "bf16", "window": 0},
        # the new token of one request, with its query
        {"name": "append_token", "kind": "append", "heads": 32, "kv": 4, "hd": 128, "n": 1, "new": 1, "rows": 300,
         "page": 16, "type": "f16", "rot": 128, "norm": True, "inter": False, "query": True},
        # a decode batch: a token of each of 32 requests, keys and values alone
        {"name": "append_lanes", "kind": "append", "heads": 32, "kv": 4, "hd": 128, "n": 32, "new": 1, "rows": 1024,
         "page": 16, "type": "bf16", "rot": 128, "norm": True, "inter": False, "query": False},
        # prompts of three requests, over four thousand tokens in all, with their queries
        {"name": "append_prompts", "kind": "append", "heads": 32, "kv": 4, "hd": 128, "n": 3, "new": 1367, "rows": 2000,
         "page": 64, "type": "f16", "rot": 128, "norm": True, "inter": False, "query": True},
        # tokens of the small dense model: no norms, neighbours paired, part of the head left as it is
        {"name": "rope_ragged", "kind": "rope", "heads": 6, "kv": 6, "hd": 48, "n": 77, "rot": 32, "norm": False,
         "inter": True, "far": 4096},
        # a prompt of 4096 tokens at far positions
        {"name": "rope_prompt", "kind": "rope", "heads": 32, "kv": 4, "hd": 128, "n": 4096, "rot": 128, "norm": True,
         "inter": False, "far": 1000000},
        # one row of the small vocabulary, five alternatives
        {"name": "logprobs_token", "kind": "logprobs", "n": 1, "vocab": 32000, "top": 5, "temper": False},
        # a decode batch over the large vocabulary at its sampling temperatures, twenty alternatives
        {"name": "logprobs_lanes", "kind": "logprobs", "n": 64, "vocab": 151936, "top": 20, "temper": True},
        # scoring a text: every row's next token, no alternatives
        {"name": "logprobs_text", "kind": "logprobs", "n": 509, "vocab": 151936, "top": 0, "temper": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((32, 4, 128), (6, 6, 48), (16, 2, 64), (8, 8, 128), (24, 8, 96), (8, 2, 256), (40, 2, 80), (28, 4, 128))


def draw(rng):
    kind = rng.choice(("attn", "attn", "append", "rope", "logprobs", "logprobs"))
    if kind == "logprobs":
        while True:
            n, vocab = _log_int(rng, 1, 512), rng.choice((32000, 151936, _log_int(rng, 1000, 151936)))
            if n * vocab <= 509 * 151936:
                return {"kind": kind, "n": n, "vocab": vocab, "top": rng.choice((0, 1, 5, 8, 20, 32)),
                        "temper": rng.random() < 0.5}
    heads, kv, hd = rng.choice(HEADS)
    rope = {"rot": rng.choice((hd, hd, hd // 4 * 2)), "norm": rng.random() < 0.6, "inter": rng.random() < 0.4}
    if kind == "rope":
        while True:
            n = _log_int(rng, 1, 4096)
            if n * (heads + kv) * hd <= 4096 * 36 * 128:
                return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "n": n, **rope, "far": _log_int(rng, 100, 1000000)}
    page, kvtype = rng.choice((16, 16, 32, 64, 128, rng.randint(1, 200))), rng.choice(sorted(DTYPES))
    while True:
        n, rows = _log_int(rng, 1, 64), _log_int(rng, 1, 65536)
        if kind == "attn":
            if n * rows * kv * hd <= 8 * 65536 * 4 * 128:
                return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "n": n, "rows": rows, "page": page,
                        "type": kvtype, "window": 0 if rng.random() < 0.75 else _log_int(rng, 1, rows)}
        else:
            rows = min(rows, 4096)
            new = rng.choice((1, 1, _log_int(rng, 1, rows)))
            if n * new * (heads + 2 * kv) * hd <= 3 * 1367 * 40 * 128 and n * rows * kv * hd <= 64 * 4096 * 4 * 128:
                return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "n": n, "new": new, "rows": rows, "page": page,
                        "type": kvtype, **rope, "query": rng.random() < 0.6}


# ---- inputs -------------------------------------------------------------------


def _lens(case):
    """Rows of every request: spread over the range, the last the longest, a prompt's new rows among them."""
    n, rows = case["n"], case["rows"]
    return [max(1, case.get("new", 1), (i + 1) * rows // n) for i in range(n)]


def _freqs(rot):
    return 1.0 / 10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.default_rng(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    s = {"case": case}
    if case["kind"] == "logprobs":
        n, V = case["n"], case["vocab"]
        s["logits"] = normal(n, V, scale=3.0)
        s["tokens"] = torch.tensor(host.integers(0, V, n), dtype=torch.int32, device="cuda")
        s["temperature"] = torch.rand(n, generator=g, device="cuda") + 0.5 if case["temper"] else None
        return s
    H, KV, hd, n = (case[k] for k in ("heads", "kv", "hd", "n"))
    if case["kind"] == "rope":
        s["q"], s["k"] = normal(n, H, hd, scale=2.0), normal(n, KV, hd, scale=2.0)
        s["pos"] = torch.tensor(host.integers(0, case["far"], n), dtype=torch.int32, device="cuda")
    else:
        dt, page = DTYPES[case["type"]], case["page"]
        lens = host.permutation(_lens(case))
        used = [-(-int(x) // page) for x in lens]
        # every request's pages lie anywhere in the pool; a table's row ends in -1
        order = host.permutation(sum(used))
        table = np.full((n, max(used)), -1, np.int32)
        at = 0
        for i, u in enumerate(used):
            table[i, :u] = order[at:at + u]
            at += u
        s["table"] = torch.tensor(table, device="cuda")
        s["k_pages"], s["v_pages"] = (normal(sum(used), page, KV, hd).to(dt) for _ in range(2))
        if case["kind"] == "attn":
            s["q"] = normal(n, H, hd)
            s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            s["scale"] = 1.0 / math.sqrt(hd)
            return s
        new = case["new"]
        T = n * new  # each request's last rows
        # queries, keys and values side by side, as one projection leaves them
        qkv = normal(T, (H + 2 * KV) * hd, scale=2.0)
        q, k, v = qkv.split((H * hd, KV * hd, KV * hd), dim=1)
        s["q"] = q.unflatten(1, (H, hd)) if case["query"] else None
        s["k"], s["v"] = k.unflatten(1, (KV, hd)), v.unflatten(1, (KV, hd))
        s["lanes"] = torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(new)
        s["pos"] = torch.tensor(np.concatenate([np.arange(x - new, x) for x in lens]), dtype=torch.int32, device="cuda")
    s["freqs"] = _freqs(case["rot"])
    s["q_norm"], s["k_norm"] = (1.0 + normal(hd, scale=0.1) if case["norm"] else None for _ in range(2))
    return s


# ---- the operators -------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _framework():
    import loom_amd
    from loom_amd import serving

    loom_amd.init(0)  # once, as a program does when it starts
    return serving


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        serving = _framework()
        if kind == "attn":
            return serving.paged_attn_dev(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"],
                                          window=case["window"])
        if kind == "append":
            q = serving.paged_append_dev(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["pos"],
                                         lanes=s["lanes"], freqs=s["freqs"], k_norm=s["k_norm"], q=s["q"],
                                         q_norm=s["q_norm"], interleaved=case["inter"])
            return (s["k_pages"], s["v_pages"]) if q is None else (s["k_pages"], s["v_pages"], q)
        if kind == "rope":
            return serving.qk_norm_rope_dev(s["q"], s["k"], s["pos"], s["freqs"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                            interleaved=case["inter"])
        out = serving.token_logprobs_dev(s["logits"], s["tokens"], top=case["top"], temperature=s["temperature"])
        return out if case["top"] else out[:2]
    return {"attn": _attn, "append": _append, "rope": _rope, "logprobs": _logprobs}[kind](s)


def _attn(s):
    q, table, lens, window = s["q"], s["table"], s["lens"], s["case"]["window"]
    n, H, hd = q.shape
    page, KV = s["k_pages"].shape[1:3]
    G, rows = H // KV, table.shape[1] * page
    at = table.clamp(min=0).long()
    k, v = (s[x][at].view(n, rows, KV, hd).float().permute(0, 2, 1, 3) for x in ("k_pages", "v_pages"))  # [n][KV][rows][hd]
    w = torch.matmul(q.view(n, KV, G, hd) * s["scale"], k.transpose(2, 3).contiguous())
    t = torch.arange(rows, device=q.device)[None, :]
    seen = t < lens[:, None]
    if window:
        seen &= t >= lens[:, None] - window
    w = w.masked_fill(~seen[:, None, None, :], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    return torch.matmul(w, v.contiguous()).view(n, H, hd)


def _turned(x, norm, s):
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * norm
    angle = s["pos"].double()[:, None] * s["freqs"]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    rot = s["case"]["rot"]
    out = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if s["case"]["inter"] else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., a] = x[..., a] * c - x[..., b] * n
    out[..., b] = x[..., b] * c + x[..., a] * n
    return out


def _rope(s):
    return _turned(s["q"], s["q_norm"], s), _turned(s["k"], s["k_norm"], s)


def _append(s):
    pos, page = s["pos"].long(), s["case"]["page"]
    at = (s["table"][s["lanes"].long(), pos // page].long(), pos % page)
    s["k_pages"][at] = _turned(s["k"], s["k_norm"], s).to(s["k_pages"].dtype)
    s["v_pages"][at] = s["v"].to(s["v_pages"].dtype)
    if s["q"] is None:
        return s["k_pages"], s["v_pages"]
    return s["k_pages"], s["v_pages"], _turned(s["q"], s["q_norm"], s)


def _logprobs(s):
    x, top = s["logits"], s["case"]["top"]
    z = x if s["temperature"] is None else x / s["temperature"][:, None]
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    lp = z - torch.log(total)
    given = lp.gather(1, s["tokens"].long()[:, None])[:, 0]
    entropy = -(e * lp).sum(-1) / total[:, 0]
    if not top:
        return given, entropy
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    return given, entropy, ids.to(torch.int32), lp.gather(1, ids)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["kind"] == "logprobs":
        return {"bytes": 4 * case["n"] * (case["vocab"] + 4 + 2 * case["top"]), "flops": 4 * case["n"] * case["vocab"]}
    H, KV, hd, n = (case[k] for k in ("heads", "kv", "hd", "n"))
    if case["kind"] == "attn":
        seen = sum(min(x, case["window"] or x) for x in _lens(case))
        return {"bytes": 2 * 2 * KV * hd * seen + 2 * 4 * n * H * hd + 4 * n + 4 * (seen // case["page"]),
                "flops": 4 * H * hd * seen}
    if case["kind"] == "rope":
        return {"bytes": 2 * 4 * n * (H + KV) * hd + 4 * n, "flops": 8 * n * (H + KV) * hd}
    T, q = n * case["new"], H if case["query"] else 0
    return {"bytes": T * hd * (8 * q + (4 + 2) * 2 * KV) + 12 * T, "flops": 8 * T * (q + KV) * hd}


# ---- the definitions in 64 bits -------------------------------------------------


def _exact_turn(x, norm, pos, freqs, inter):
    x = x.double()
    if norm is not None:
        x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * norm.double()
    angle = pos.double()[:, None] * freqs
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    half = len(freqs)
    part = x[..., :2 * half]
    pairs = part.unflatten(-1, (half, 2)) if inter else part.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if not inter:
        z = z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), x[..., 2 * half:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        x = s["logits"].double()
        z = x if s["temperature"] is None else x / s["temperature"].double()[:, None]
        lp = torch.log_softmax(z, -1)
        given = lp[torch.arange(case["n"]), s["tokens"].long()]
        entropy = -(lp.exp() * lp).sum(-1)
        if not case["top"]:
            return given, entropy
        return given, entropy, None, lp.topk(case["top"], -1)[0]
    if case["kind"] == "rope":
        return tuple(_exact_turn(s[x], s[x + "_norm"], s["pos"], s["freqs"], case["inter"]) for x in ("q", "k"))
    page = case["page"]
    if case["kind"] == "append":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k = _exact_turn(s["k"], s["k_norm"], s["pos"], s["freqs"], case["inter"])
        pos, lanes = s["pos"].tolist(), s["lanes"].tolist()
        table = s["table"].tolist()
        row = torch.tensor([table[i][p // page] * page + p % page for i, p in zip(lanes, pos)], device="cuda")
        k_pages.view(-1, *k.shape[1:])[row] = k
        v_pages.view(-1, *k.shape[1:])[row] = s["v"].double()
        if s["q"] is None:
            return k_pages, v_pages
        return k_pages, v_pages, _exact_turn(s["q"], s["q_norm"], s["pos"], s["freqs"], case["inter"])
    q = s["q"].double()
    n, H, hd = q.shape
    G = H // case["kv"]
    out = torch.zeros_like(q)
    for i in range(n):
        end = int(s["lens"][i])
        start = max(0, end - case["window"]) if case["window"] else 0
        t = torch.arange(start, end, device=q.device)
        at = s["table"][i].long()[t // page], t % page
        k, v = s["k_pages"][at].double(), s["v_pages"][at].double()
        for h in range(case["kv"]):
            mine = slice(h * G, (h + 1) * G)
            out[i, mine] = torch.softmax(q[i, mine] @ k[:, h].T * s["scale"], -1) @ v[:, h]
    return out
