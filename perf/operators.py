"""The operators of a batched serving step as measurable cases: attention of a
batch that shares a long prefix, the low-rank adapters of many requests beside
one projection, the target's token probabilities, and the verification of
drafted tokens against them.

`run` computes each in its plain form (elementary torch operations in 32 bits,
64 where a sampled token hangs on the last bit), or, where `own` is set,
through loom_amd.serving.  Sizes are those of the repository's own
configurations (the Qwen3-30B-A3B and stories15M shapes: heads, head size,
projections, vocabularies, the 4096-token context, 32 and 64 lanes) or generic
ragged ones.
"""
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request behind a short system prompt, one token: the latency of a call
        {"name": "attn_token", "kind": "attn", "heads": 32, "kv": 4, "hd": 128, "prefix": 256, "n": 1, "nq": 1,
         "own": 16, "ragged": False},
        # the small dense model's heads (no sharing of key heads), odd sizes, drafts of unequal lengths
        {"name": "attn_ragged", "kind": "attn", "heads": 6, "kv": 6, "hd": 48, "prefix": 1003, "n": 5, "nq": 3,
         "own": 77, "ragged": True},
        # ordinary batched decode: 32 requests behind one 4096-token prompt, a token each
        {"name": "attn_lanes", "kind": "attn", "heads": 32, "kv": 4, "hd": 128, "prefix": 4096, "n": 32, "nq": 1,
         "own": 512, "ragged": False},
        # a verification step: 64 requests, four drafted tokens and the last one, behind a long document
        {"name": "attn_drafts", "kind": "attn", "heads": 32, "kv": 4, "hd": 128, "prefix": 16384, "n": 64, "nq": 5,
         "own": 640, "ragged": True},
        # one request's adapter on the query projection, one token
        {"name": "lora_token", "kind": "lora", "n": 1, "rows": 4096, "cols": 2048, "rank": 16, "adapters": 8,
         "type": "f16", "spans": False},
        # a decode batch: every request its own adapter (some none) on the attention output projection
        {"name": "lora_lanes", "kind": "lora", "n": 32, "rows": 2048, "cols": 4096, "rank": 64, "adapters": 24,
         "type": "bf16", "spans": False},
        # odd sizes and f32 adapters, tokens of several requests mixed
        {"name": "lora_ragged", "kind": "lora", "n": 77, "rows": 1003, "cols": 1410, "rank": 9, "adapters": 5,
         "type": "f32", "spans": False},
        # prefill: the prompts of several requests, each with its adapter, through the query projection
        {"name": "lora_prefill", "kind": "lora", "n": 2048, "rows": 4096, "cols": 2048, "rank": 32, "adapters": 12,
         "type": "f16", "spans": True},
        # one row of the small vocabulary
        {"name": "probs_token", "kind": "probs", "rows": 1, "vocab": 32000},
        # the rows of a verification step over the large vocabulary
        {"name": "probs_drafts", "kind": "probs", "rows": 160, "vocab": 151936},
        # one request, three drafted tokens that came without probabilities (a greedy drafter)
        {"name": "verify_token", "kind": "verify", "n": 1, "k": 3, "vocab": 32000, "greedy": True},
        # 64 requests with four drafted tokens each (some fewer) over the large vocabulary
        {"name": "verify_drafts", "kind": "verify", "n": 64, "k": 4, "vocab": 151936, "greedy": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "lora", "lora", "probs", "verify"))
    if kind == "attn":
        heads, kv, hd = rng.choice(((32, 4, 128), (6, 6, 48), (16, 2, 64), (8, 8, 128), (24, 8, 96), (8, 2, 256)))
        while True:
            prefix, n, nq, own_rows = _log_int(rng, 1, 16384), _log_int(rng, 1, 64), rng.randint(1, 6), _log_int(rng, 8, 1024)
            if heads * n * nq * (prefix + own_rows) * hd <= 32 * 64 * 5 * (16384 + 640) * 128:
                return {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "prefix": prefix, "n": n, "nq": nq,
                        "own": own_rows, "ragged": rng.random() < 0.5}
    if kind == "lora":
        n, rows, cols = _log_int(rng, 1, 2048), _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
        if rng.random() < 0.5:
            rows, cols = (rows + 63) // 64 * 64, (cols + 63) // 64 * 64
        while n * (rows + cols) > 2048 * 6144:
            n //= 2
        return {"kind": kind, "n": n, "rows": rows, "cols": cols, "rank": rng.choice((1, 4, 8, 16, 24, 32, 64)),
                "adapters": rng.randint(1, 32), "type": rng.choice(sorted(DTYPES)), "spans": n >= 64 and rng.random() < 0.7}
    vocab = rng.choice((32000, 151936, _log_int(rng, 1000, 151936)))
    if kind == "probs":
        return {"kind": kind, "rows": _log_int(rng, 1, 160), "vocab": vocab}
    return {"kind": kind, "n": _log_int(rng, 1, 64), "k": rng.randint(1, 4), "vocab": vocab, "greedy": rng.random() < 0.3}


# ---- inputs -------------------------------------------------------------------


def _lens(case):
    """Rows of every request's own cache, its query rows included: spread over the range, the last the longest."""
    n, nq, rows = case["n"], case["nq"], case["own"]
    return [max(min(nq, rows), (i + 1) * rows // n) for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.default_rng(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    s = {"case": case}
    if case["kind"] == "attn":
        H, KV, hd, P, n, nq, rows = (case[k] for k in ("heads", "kv", "hd", "prefix", "n", "nq", "own"))
        # caches as the decode frame holds them: fp16 rows of every key head; keys after QK-norm and rope have
        # unit-sized elements, so the scores spread over several units
        s["q"] = normal(n, nq, H, hd)
        s["k_prefix"], s["v_prefix"] = normal(P, KV, hd).half(), normal(P, KV, hd).half()
        s["k_own"], s["v_own"] = normal(n, rows, KV, hd).half(), normal(n, rows, KV, hd).half()
        s["own_len"] = torch.tensor(host.permutation(_lens(case)), dtype=torch.int32, device="cuda")
        s["q_len"] = None
        if case["ragged"]:
            s["q_len"] = torch.tensor(host.permutation([1 + i % nq for i in range(n)]), dtype=torch.int32, device="cuda")
        s["scale"] = 1.0 / math.sqrt(hd)
    elif case["kind"] == "lora":
        n, rows, cols, r, E = (case[k] for k in ("n", "rows", "cols", "rank", "adapters"))
        dt = DTYPES[case["type"]]
        s["x"], s["base"] = normal(n, cols), normal(n, rows)
        s["a"] = normal(E, r, cols, scale=1.0 / math.sqrt(cols)).to(dt)
        s["b"] = normal(E, rows, r, scale=1.0 / math.sqrt(r)).to(dt)
        s["scale"] = torch.rand(E, generator=g, device="cuda") + 0.5
        if case["spans"]:  # each request's tokens follow one another
            ids = np.repeat(host.integers(-1, E, 8), -(-n // 8))[:n]
        else:
            ids = host.integers(-1, E, n)
        if n == 1:
            ids[:] = host.integers(0, E)
        s["ids"] = torch.tensor(ids, dtype=torch.int32, device="cuda")
    elif case["kind"] == "probs":
        s["logits"] = normal(case["rows"], case["vocab"], scale=3.0)
        s["temperature"] = torch.rand(case["rows"], generator=g, device="cuda") + 0.5
    else:
        n, k, V = case["n"], case["k"], case["vocab"]
        logits = normal(n, k + 1, V, scale=3.0)
        s["target"] = torch.softmax(logits, -1)
        near = torch.softmax(logits[:, :k] + normal(n, k, V, scale=0.5), -1)
        if case["greedy"]:
            s["draft"], s["tokens"] = None, near.argmax(-1).to(torch.int32)
        else:
            s["draft"] = near
            s["tokens"] = torch.multinomial(near.view(n * k, V), 1, generator=g).view(n, k).to(torch.int32)
        s["u_accept"] = torch.rand(n, k, generator=g, device="cuda")
        s["u_sample"] = torch.rand(n, generator=g, device="cuda")
        s["n_draft"] = torch.tensor(host.permutation([k - i % 2 if n > 1 else k for i in range(n)]), dtype=torch.int32,
                                    device="cuda")
    return s


# ---- the operators -------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _framework():
    import loom_amd
    from loom_amd import serving

    loom_amd.init(0)  # once, as a program does when it starts
    return serving


def run(s):
    kind = s["case"]["kind"]
    if own:
        serving = _framework()
        if kind == "attn":
            return serving.prefix_attn_dev(s["q"], s["k_prefix"], s["v_prefix"], s["k_own"], s["v_own"], s["own_len"],
                                           s["scale"], q_len=s["q_len"])
        if kind == "lora":
            return serving.lora_dev(s["x"], s["a"], s["b"], s["scale"], s["ids"], base=s["base"])
        if kind == "probs":
            return serving.token_probs_dev(s["logits"], s["temperature"])
        return serving.verify_drafts_dev(s["target"], s["tokens"], s["u_accept"], s["u_sample"], draft_probs=s["draft"],
                                         n_draft=s["n_draft"])
    return {"attn": _attn, "lora": _lora, "probs": _probs, "verify": _verify}[kind](s)


def _attn(s):
    q, own_len, q_len = s["q"], s["own_len"], s["q_len"]
    n, nq, H, hd = q.shape
    P, KV = s["k_prefix"].shape[:2]
    rows, G = s["k_own"].shape[1], H // KV
    qk = q.view(n, nq, KV, G, hd).permute(2, 0, 1, 3, 4) * s["scale"]  # [KV][n][nq][G][hd]
    kp, vp = (s[x].float().permute(1, 0, 2) for x in ("k_prefix", "v_prefix"))  # [KV][P][hd]
    ko, vo = (s[x].float().permute(2, 0, 1, 3) for x in ("k_own", "v_own"))  # [KV][n][rows][hd]
    shared = torch.matmul(qk.reshape(KV, n * nq * G, hd), kp.transpose(1, 2).contiguous()).view(KV, n, nq * G, P)
    mine = torch.matmul(qk.reshape(KV, n, nq * G, hd), ko.transpose(2, 3).contiguous())
    # query j of a request with L of them sees its own rows up to its own: own_len - L + j
    L = torch.full_like(own_len, nq) if q_len is None else q_len
    j = torch.arange(nq, device=q.device)
    seen = own_len[:, None] - L[:, None] + 1 + j[None, :]  # [n][nq]
    mask = torch.arange(rows, device=q.device)[None, None, :] < seen[:, :, None]  # [n][nq][rows]
    mine = mine.view(KV, n, nq, G, rows).masked_fill(~mask[None, :, :, None, :], -math.inf).view(KV, n, nq * G, rows)
    w = torch.cat([shared, mine], -1)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    out = torch.matmul(w[..., :P].reshape(KV, n * nq * G, P), vp.contiguous()).view(KV, n, nq * G, hd)
    out = out + torch.matmul(w[..., P:].contiguous(), vo.contiguous())
    out = out.view(KV, n, nq, G, hd).permute(1, 2, 0, 3, 4).reshape(n, nq, H, hd)
    return out.masked_fill((j[None, :] >= L[:, None])[:, :, None, None], 0.0)


def _lora(s):
    x, ids = s["x"], s["ids"]
    E, r, cols = s["a"].shape
    rows = s["b"].shape[1]
    # every adapter's product, and of them each token's own
    y = torch.matmul(x, s["a"].float().view(E * r, cols).t().contiguous()).view(-1, E, r)
    mine = torch.arange(E, device=x.device)[None, :] == ids[:, None]
    y = torch.where(mine[:, :, None], y * s["scale"][None, :, None], torch.zeros_like(y))
    return s["base"] + torch.matmul(y.view(-1, E * r), s["b"].float().permute(0, 2, 1).reshape(E * r, rows))


def _probs(s):
    z = s["logits"] / s["temperature"][:, None]
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _verify(s):
    # in 64 bits: a product at the border of acceptance and a running sum next to the drawn number decide a token
    target, tok, n_draft = s["target"], s["tokens"].long(), s["n_draft"]
    n, k = tok.shape
    px = target[:, :k].gather(2, tok[:, :, None])[:, :, 0].double()
    qx = torch.ones_like(px) if s["draft"] is None else s["draft"].gather(2, tok[:, :, None])[:, :, 0].double()
    ok = (s["u_accept"].double() * qx < px) & (torch.arange(k, device=tok.device)[None, :] < n_draft[:, None])
    accepted = ok.long().cumprod(1).sum(1)  # [n]
    lane = torch.arange(n, device=tok.device)
    p = target[lane, accepted].double()
    rejected = accepted < n_draft
    at = accepted.clamp(max=k - 1)
    if s["draft"] is None:
        q = torch.zeros_like(p)
        q[lane, tok[lane, at]] = math.inf
    else:
        q = s["draft"][lane, at].double()
    d = (p - torch.where(rejected[:, None], q, torch.zeros_like(q))).clamp(min=0.0)
    d = torch.where(d.sum(1, keepdim=True) > 0, d, p)
    c = d.cumsum(1)
    last = (c <= s["u_sample"].double()[:, None] * c[:, -1:]).sum(1)
    j = torch.arange(k + 1, device=tok.device)[None, :]
    out = torch.where(j < accepted[:, None], torch.cat([tok, tok[:, -1:]], 1), torch.full((n, k + 1), -1, device=tok.device))
    out = torch.where(j == accepted[:, None], last[:, None], out)
    return out.to(torch.int32), accepted.to(torch.int32)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["kind"] == "attn":
        H, KV, hd, P, n, nq = (case[k] for k in ("heads", "kv", "hd", "prefix", "n", "nq"))
        lens = _lens(case)
        live = [1 + i % nq for i in range(n)] if case["ragged"] else [nq] * n
        cache = 2 * KV * hd * 2 * (P + sum(lens))
        flops = 4 * H * hd * (P * sum(live) + sum(lens) * sum(live) / n)
        return {"bytes": cache + 2 * 4 * H * hd * sum(live) + 4 * n, "flops": flops}
    if case["kind"] == "lora":
        n, rows, cols, r, E = (case[k] for k in ("n", "rows", "cols", "rank", "adapters"))
        size = 4 if case["type"] == "f32" else 2
        used = min(E, 8) if case["spans"] else E * (1 - (1 - 1 / (E + 1)) ** n) if n > 1 else 1
        return {"bytes": 4 * n * (cols + 2 * rows) + size * used * r * (rows + cols) + 4 * n,
                "flops": 2 * n * r * (rows + cols)}
    if case["kind"] == "probs":
        return {"bytes": 8 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}
    n, k, V = case["n"], case["k"], case["vocab"]
    # the target's row of the sampled token, the drafter's beside it, a few values of the others
    return {"bytes": n * V * 4 * (1 if case["greedy"] else 2) + n * k * 20, "flops": 2 * n * V}


# ---- the definitions in 64 bits -------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attn":
        q = s["q"].double()
        n, nq, H, hd = q.shape
        G = H // case["kv"]
        out = torch.zeros_like(q)
        for i in range(n):
            L = nq if s["q_len"] is None else int(s["q_len"][i])
            rows = int(s["own_len"][i])
            for h in range(case["kv"]):
                k = torch.cat([s["k_prefix"][:, h], s["k_own"][i, :rows, h]]).double()
                v = torch.cat([s["v_prefix"][:, h], s["v_own"][i, :rows, h]]).double()
                for j in range(L):
                    end = len(k) - L + 1 + j
                    qj = q[i, j, h * G:(h + 1) * G]
                    p = torch.softmax(qj @ k[:end].T * s["scale"], -1)
                    out[i, j, h * G:(h + 1) * G] = p @ v[:end]
        return out
    if case["kind"] == "lora":
        x, out = s["x"].double(), s["base"].double().clone()
        for e in range(case["adapters"]):
            at = (s["ids"] == e).nonzero()[:, 0]
            out[at] += s["scale"][e].double() * ((x[at] @ s["a"][e].double().T) @ s["b"][e].double().T)
        return out
    if case["kind"] == "probs":
        return torch.softmax(s["logits"].double() / s["temperature"].double()[:, None], -1)
    return None  # tokens and counts: whole numbers, held to the plain form's
