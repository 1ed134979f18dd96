"""Batched serving on the device: what a server with many requests of one
model runs between the projections and the next token.

* ``prefix_attn_dev`` -- attention of a batch that shares a prefix, the prefix
  read once for all lanes, each lane's own rows beside it;
* ``lora_dev`` -- the low-rank adapters of many requests beside one projection;
* ``token_probs_dev`` -- probabilities from logits at a temperature;
* ``verify_drafts_dev`` -- drafted tokens against the target's probabilities.

Tensors are torch device tensors on the current device, which is the one
``loom_amd.init`` was given; the calls run on torch's current stream, take
their outputs and workspace from torch's allocator, never wait for the device
and can be captured in a graph.  They are inference operators: no gradient is
recorded.  Wrong shapes, types or devices raise ``ValueError``, what the
library refuses or does not serve ``LoomHipError``.
"""
from __future__ import annotations

import ctypes as C

from . import BF16, F16, F32, KvRowsDesc, LoomHipError, LoraDesc, OK, last_error, lib
from .backend import _stream

_LORA_TYPES = {}


def _torch():
    import torch

    return torch


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on_device(**tensors) -> None:
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} is on {t.device}, not on the GPU")
        if dev is None:
            dev = _torch().cuda.current_device()
        if t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, the current device is {dev}")


def _run(rc: int, what: str) -> None:
    """These calls have no path of the caller's to fall back to: a decline is an error too."""
    if rc != OK:
        raise LoomHipError(f"{what}: {last_error()} (rc={rc})")


def _ws(n: int, like):
    """A workspace of n bytes from torch's allocator, or None."""
    return _torch().empty(n, dtype=_torch().uint8, device=like.device) if n else None


def _p(t):
    return None if t is None else t.data_ptr()


def _kv_desc(k, v, lanes: bool, name: str):
    torch = _torch()
    want = 4 if lanes else 3
    _need(k.dim() == want and k.shape == v.shape and (k.stride() == v.stride() or k.numel() == 0),
          f"{name}: keys and values of one shape and layout, [{'n, ' if lanes else ''}rows, n_kv_heads, head_dim]")
    _need(k.dtype == v.dtype and k.dtype in (torch.float16, torch.int16), f"{name}: fp16 rows (or their bits as int16)")
    if k.numel() == 0:
        return KvRowsDesc()
    _need(k.stride(-1) == 1 or k.shape[-1] == 1, f"{name}: the values of a head one after the other")
    return KvRowsDesc(k.data_ptr(), v.data_ptr(), k.shape[-3], k.stride(0) if lanes else 0, k.stride(-3), k.stride(-2))


def prefix_attn_dev(q, k_prefix, v_prefix, k_own, v_own, own_len, scale: float, q_len=None, out=None):
    """Attention of n lanes over a shared prefix and their own rows.

    q f32 [n, n_q, n_heads, head_dim]; k_prefix, v_prefix fp16 [prefix, n_kv_heads, head_dim] (None: no prefix);
    k_own, v_own fp16 [n, rows, n_kv_heads, head_dim] (None: none), of which lane i holds own_len[i] (int32), the last
    q_len[i] of them its query tokens' own (int32; None: n_q each).  Caches of any row, head and lane strides that are
    multiples of 8, a ``Decoder``'s at one layer among them.  Returns out f32 as q; rows past q_len[i] keep what an
    ``out`` given holds, and are zero in one made here.
    """
    torch = _torch()
    _need(q.dim() == 4 and q.dtype == torch.float32 and q.is_contiguous(), "q: contiguous f32 [n, n_q, n_heads, head_dim]")
    n, n_q, heads, hd = q.shape
    pre, own = KvRowsDesc(), KvRowsDesc()
    kv = None
    if k_prefix is not None:
        pre = _kv_desc(k_prefix, v_prefix, False, "prefix")
        kv = k_prefix.shape[-2]
        _need(k_prefix.shape[-1] == hd, "prefix: another head size than q's")
    if k_own is not None:
        own = _kv_desc(k_own, v_own, True, "own")
        _need(k_own.shape[0] == n and k_own.shape[-1] == hd and kv in (None, k_own.shape[-2]),
              "own: lanes and head size as q's, key heads as the prefix's")
        _need(own_len is not None, "own rows without own_len")
        kv = k_own.shape[-2]
    _need(kv is not None, "neither a prefix nor own rows")
    for name, t in (("own_len", own_len), ("q_len", q_len)):
        _need(t is None or (t.dtype == torch.int32 and t.shape == (n,) and t.is_contiguous()), f"{name}: int32 [n]")
    if out is None:
        out = torch.empty_like(q) if q_len is None else torch.zeros_like(q)
    _need(out.shape == q.shape and out.dtype == torch.float32 and out.is_contiguous(), "out: as q")
    _on_device(q=q, k_prefix=k_prefix, v_prefix=v_prefix, k_own=k_own, v_own=v_own, own_len=own_len, q_len=q_len, out=out)
    L = lib()
    ws = L.loomhip_prefix_attn_ws(pre.rows, own.rows, n, n_q, heads, kv, hd)
    w = _ws(ws, q)
    _run(L.loomhip_prefix_attn_dev(C.byref(pre), C.byref(own), _p(q), _p(own_len), _p(q_len), n, n_q, heads, kv, hd,
                                   scale, _p(out), _p(w), ws, _stream()), "prefix_attn_dev")
    return out


def lora_dev(x, a, b, scale, ids, base=None, out=None):
    """out[t] = base[t] + scale[e] * b[e] @ (a[e] @ x[t]) with e = ids[t]; base[t] alone where ids[t] is no adapter.

    x f32 [n, cols], a [adapters, rank, cols] and b [adapters, rows, rank] of one type (f32, fp16, bf16), scale f32
    [adapters], ids int32 [n], base f32 [n, rows] or None (zeros).  ``out=base`` adds in place, as beside
    ``matvec_dev``'s output.  Rows of x, base and out may be strided.  Returns out.
    """
    torch = _torch()
    if not _LORA_TYPES:
        _LORA_TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    _need(x.dim() == 2 and x.dtype == torch.float32, "x: f32 [n, cols]")
    _need(a.dim() == 3 and b.dim() == 3 and a.dtype == b.dtype and a.dtype in _LORA_TYPES and a.is_contiguous()
          and b.is_contiguous(), "a, b: contiguous, of one type (f32, fp16 or bf16)")
    n, cols = x.shape
    adapters, rank = a.shape[:2]
    rows = b.shape[1]
    _need(a.shape[2] == cols and b.shape[0] == adapters and b.shape[2] == rank,
          "a [adapters, rank, cols], b [adapters, rows, rank]")
    _need(scale.shape == (adapters,) and scale.dtype == torch.float32 and scale.is_contiguous(), "scale: f32 [adapters]")
    _need(ids.shape == (n,) and ids.dtype == torch.int32 and ids.is_contiguous(), "ids: int32 [n]")
    if out is None:
        out = torch.empty((n, rows), dtype=torch.float32, device=x.device)
    for name, t, w in (("x", x, cols), ("base", base, rows), ("out", out, rows)):
        _need(t is None or (t.shape == (n, w) and t.dtype == torch.float32 and (w == 1 or t.stride(1) == 1)
                            and (n == 1 or t.stride(0) >= w)), f"{name}: f32 [{n}, {w}], rows of consecutive values")
    _on_device(x=x, a=a, b=b, scale=scale, ids=ids, base=base, out=out)
    L = lib()
    d = LoraDesc(_LORA_TYPES[a.dtype], adapters, rank, rows, cols, a.data_ptr(), b.data_ptr(), scale.data_ptr())
    ws = L.loomhip_lora_ws(C.byref(d), n)
    w = _ws(ws, x)
    _run(L.loomhip_lora_dev(C.byref(d), _p(x), max(x.stride(0), cols), _p(ids), _p(base),
                            max(base.stride(0), rows) if base is not None else rows, n, _p(out),
                            max(out.stride(0), rows), _p(w), ws, _stream()), "lora_dev")
    return out


def token_probs_dev(logits, temperature=None, out=None):
    """softmax(logits / temperature) of every row: logits f32 [..., vocab] contiguous, temperature f32 of the leading
    shape (None: 1; not positive: 1 at the first maximum).  ``out=logits`` works in place.  Returns out."""
    torch = _torch()
    _need(logits.dim() >= 1 and logits.dtype == torch.float32 and logits.is_contiguous(), "logits: contiguous f32")
    vocab = logits.shape[-1]
    n = logits.numel() // vocab if vocab else 0
    _need(temperature is None or (temperature.dtype == torch.float32 and temperature.shape == logits.shape[:-1]
                                  and temperature.is_contiguous()), "temperature: f32, one a row")
    if out is None:
        out = torch.empty_like(logits)
    _need(out.shape == logits.shape and out.dtype == torch.float32 and out.is_contiguous(), "out: as logits")
    _on_device(logits=logits, temperature=temperature, out=out)
    L = lib()
    ws = L.loomhip_token_probs_ws(n, vocab)
    w = _ws(ws, logits)
    _run(L.loomhip_token_probs_dev(_p(logits), n, vocab, vocab, _p(temperature), _p(out), vocab, _p(w), ws, _stream()),
         "token_probs_dev")
    return out


def verify_drafts_dev(target_probs, draft_tokens, u_accept, u_sample, draft_probs=None, n_draft=None):
    """Drafted tokens against the target's probabilities, from given random numbers in [0, 1).

    target_probs f32 [n, k + 1, vocab], draft_tokens int32 [n, k], u_accept f32 [n, k], u_sample f32 [n], draft_probs
    f32 [n, k, vocab] (None: a drafter that names one token), n_draft int32 [n] (None: k each).  Returns (tokens int32
    [n, k + 1]: the accepted ones, the next one, then -1; accepted int32 [n]).
    """
    torch = _torch()
    _need(target_probs.dim() == 3 and target_probs.shape[1] >= 1, "target_probs: f32 [n, k + 1, vocab]")
    n, k1, vocab = target_probs.shape
    k = k1 - 1
    for name, t, shape, dt in (("target_probs", target_probs, (n, k1, vocab), torch.float32),
                               ("draft_tokens", draft_tokens, (n, k), torch.int32),
                               ("u_accept", u_accept, (n, k), torch.float32), ("u_sample", u_sample, (n,), torch.float32),
                               ("draft_probs", draft_probs, (n, k, vocab), torch.float32),
                               ("n_draft", n_draft, (n,), torch.int32)):
        _need(t is None or (t.shape == shape and t.dtype == dt and t.is_contiguous()),
              f"{name}: contiguous {str(dt)[6:]} {list(shape)}")
    _on_device(target_probs=target_probs, draft_tokens=draft_tokens, u_accept=u_accept, u_sample=u_sample,
               draft_probs=draft_probs, n_draft=n_draft)
    tokens = torch.empty((n, k1), dtype=torch.int32, device=target_probs.device)
    accepted = torch.empty((n,), dtype=torch.int32, device=target_probs.device)
    L = lib()
    ws = L.loomhip_verify_drafts_ws(n, vocab)
    w = _ws(ws, target_probs)
    _run(L.loomhip_verify_drafts_dev(_p(target_probs), _p(draft_probs), _p(draft_tokens), _p(n_draft), _p(u_accept),
                                     _p(u_sample), n, k, vocab, _p(tokens), _p(accepted), _p(w), ws, _stream()),
         "verify_drafts_dev")
    return tokens, accepted


__all__ = ["lora_dev", "prefix_attn_dev", "token_probs_dev", "verify_drafts_dev"]
