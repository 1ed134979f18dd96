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
import functools

import torch

from . import BF16, F16, F32, KvRowsDesc, LoomHipError, LoraDesc, OK, last_error, lib

_F32, _I32, _U8 = torch.float32, torch.int32, torch.uint8
_LORA_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_HALF = (torch.float16, torch.int16)

# A serving step makes hundreds of these calls, each a few microseconds of device work: the checks below are plain
# comparisons, messages are formed only when one fails, and workspace sizes are remembered by the sizes they follow from.


def _place(first, *others) -> tuple:
    """(device, stream handle) for tensors that have to be on the current device; raises ValueError otherwise."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    if dev < 0:
        raise ValueError(f"tensors on {first.device}, not on the GPU")
    if dev != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on {first.device}, the current device is {torch.cuda.current_device()}")
    return first.device, torch._C._cuda_getCurrentRawStream(dev)


def _fail(what: str, rc: int):
    """These calls have no path of the caller's to fall back to: a decline is an error too."""
    raise LoomHipError(f"{what}: {last_error()} (rc={rc})")


@functools.lru_cache(maxsize=4096)
def _attn_ws(*sizes) -> int:
    return lib().loomhip_prefix_attn_ws(*sizes)


@functools.lru_cache(maxsize=4096)
def _lora_ws(n: int, t: int, *sizes) -> int:
    return lib().loomhip_lora_ws(C.byref(LoraDesc(t, *sizes)), n)


@functools.lru_cache(maxsize=4096)
def _probs_ws(n: int, vocab: int) -> int:
    return lib().loomhip_token_probs_ws(n, vocab)


@functools.lru_cache(maxsize=4096)
def _verify_ws(n: int, vocab: int) -> int:
    return lib().loomhip_verify_drafts_ws(n, vocab)


_NO_ROWS = KvRowsDesc()


def _kv_desc(k, v, lanes: bool, name: str):
    shape, stride = k.shape, k.stride()
    if (len(shape) != 3 + lanes or v.shape != shape or k.dtype not in _HALF or v.dtype != k.dtype):
        raise ValueError(f"{name}: keys and values of one shape, [{'n, ' if lanes else ''}rows, n_kv_heads, head_dim], fp16 "
                         "(or its bits as int16)")
    if 0 in shape:
        return _NO_ROWS
    if (v.stride() != stride and any(a != b for a, b, s in zip(stride, v.stride(), shape) if s > 1)) or (
            stride[-1] != 1 and shape[-1] != 1):
        raise ValueError(f"{name}: keys and values of one layout, the values of a head one after the other")
    return KvRowsDesc(k.data_ptr(), v.data_ptr(), shape[-3], stride[0] if lanes else 0, stride[-3], stride[-2])


def prefix_attn_dev(q, k_prefix, v_prefix, k_own, v_own, own_len, scale: float, q_len=None, out=None):
    """Attention of n lanes over a shared prefix and their own rows.

    q f32 [n, n_q, n_heads, head_dim]; k_prefix, v_prefix fp16 [prefix, n_kv_heads, head_dim] (None: no prefix);
    k_own, v_own fp16 [n, rows, n_kv_heads, head_dim] (None: none), of which lane i holds own_len[i] (int32), the last
    q_len[i] of them its query tokens' own (int32; None: n_q each).  Caches of any row, head and lane strides that are
    multiples of 8, a ``Decoder``'s at one layer among them; the work is cut by `rows`, so pass what the longest lane holds
    (a view) rather than a cache's whole length.  Returns out f32 as q; rows past q_len[i] keep what an
    ``out`` given holds, and are zero in one made here.
    """
    shape = q.shape
    if len(shape) != 4 or q.dtype is not _F32 or not q.is_contiguous():
        raise ValueError("q: contiguous f32 [n, n_q, n_heads, head_dim]")
    n, n_q, heads, hd = shape
    if (k_prefix is None) != (v_prefix is None) or (k_own is None) != (v_own is None):
        raise ValueError("keys without values, or values without keys")
    pre = own = _NO_ROWS
    kv = None
    if k_prefix is not None:
        pre = _kv_desc(k_prefix, v_prefix, False, "prefix")
        kv = k_prefix.shape[1]
        if k_prefix.shape[2] != hd:
            raise ValueError("prefix: another head size than q's")
    if k_own is not None:
        own = _kv_desc(k_own, v_own, True, "own")
        s = k_own.shape
        if s[0] != n or s[3] != hd or (kv is not None and s[2] != kv):
            raise ValueError("own: lanes and head size as q's, key heads as the prefix's")
        kv = s[2]
        if own_len is None:
            raise ValueError("own rows without own_len")
    elif k_prefix is None:
        raise ValueError("neither a prefix nor own rows")
    for t in (own_len, q_len):
        if t is not None and (t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous()):
            raise ValueError("own_len, q_len: int32 [n]")
    dev, stream = _place(q, k_prefix, v_prefix, k_own, v_own, own_len, q_len, out)
    fresh = out is None
    if fresh:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not _F32 or not out.is_contiguous():
        raise ValueError("out: as q")
    nb = _attn_ws(pre.rows, own.rows, n, n_q, heads, kv, hd)
    ws = torch.empty(nb, dtype=_U8, device=dev) if nb else None
    rc = lib().loomhip_prefix_attn_dev(
        C.byref(pre), C.byref(own), q.data_ptr(), None if own_len is None else own_len.data_ptr(),
        None if q_len is None else q_len.data_ptr(), n, n_q, heads, kv, hd, scale, out.data_ptr(), fresh,
        ws.data_ptr() if nb else None, nb, stream)
    if rc != OK:
        _fail("prefix_attn_dev", rc)
    return out


def _rows_ok(t, n: int, width: int) -> bool:
    """f32 [n, width] whose rows are consecutive values and do not overlap."""
    return (t.shape == (n, width) and t.dtype is _F32 and (t.is_contiguous() or (
        (width == 1 or t.stride(1) == 1) and (n == 1 or t.stride(0) >= width))))


def lora_dev(x, a, b, scale, ids, base=None, out=None):
    """out[t] = base[t] + scale[e] * b[e] @ (a[e] @ x[t]) with e = ids[t]; base[t] alone where ids[t] is no adapter.

    x f32 [n, cols], a [adapters, rank, cols] and b [adapters, rows, rank] of one type (f32, fp16, bf16), scale f32
    [adapters], ids int32 [n], base f32 [n, rows] or None (zeros).  ``out=base`` adds in place, as beside
    ``matvec_dev``'s output.  Rows of x, base and out may be strided.  Returns out.
    """
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError("x [n, cols], a [adapters, rank, cols], b [adapters, rows, rank]")
    n, cols = x.shape
    adapters, rank, ac = a.shape
    rows = b.shape[1]
    kind = _LORA_TYPES.get(a.dtype)
    if kind is None or b.dtype != a.dtype or not a.is_contiguous() or not b.is_contiguous():
        raise ValueError("a, b: contiguous, of one type (f32, fp16 or bf16)")
    if ac != cols or b.shape[0] != adapters or b.shape[2] != rank:
        raise ValueError("a [adapters, rank, cols], b [adapters, rows, rank]")
    if scale.shape != (adapters,) or scale.dtype is not _F32 or not scale.is_contiguous():
        raise ValueError("scale: f32 [adapters]")
    if ids.shape != (n,) or ids.dtype is not _I32 or not ids.is_contiguous():
        raise ValueError("ids: int32 [n]")
    dev, stream = _place(x, a, b, scale, ids, base, out)
    if out is None:
        out = torch.empty((n, rows), dtype=_F32, device=dev)
    if not _rows_ok(x, n, cols) or not _rows_ok(out, n, rows) or not (base is None or _rows_ok(base, n, rows)):
        raise ValueError("x [n, cols], base and out [n, rows]: f32, rows of consecutive values")
    nb = _lora_ws(n, kind, adapters, rank, rows, cols)
    ws = torch.empty(nb, dtype=_U8, device=dev) if nb else None
    d = LoraDesc(kind, adapters, rank, rows, cols, a.data_ptr(), b.data_ptr(), scale.data_ptr())
    rc = lib().loomhip_lora_dev(
        C.byref(d), x.data_ptr(), x.stride(0) if n > 1 else cols, ids.data_ptr(), None if base is None else base.data_ptr(),
        base.stride(0) if base is not None and n > 1 else rows, n, out.data_ptr(), out.stride(0) if n > 1 else rows,
        ws.data_ptr() if nb else None, nb, stream)
    if rc != OK:
        _fail("lora_dev", rc)
    return out


def token_probs_dev(logits, temperature=None, out=None):
    """softmax(logits / temperature) of every row: logits f32 [..., vocab] contiguous, temperature f32 of the leading
    shape (None: 1; not positive: 1 at the first maximum).  ``out=logits`` works in place.  Returns out."""
    shape = logits.shape
    if not shape or logits.dtype is not _F32 or not logits.is_contiguous():
        raise ValueError("logits: contiguous f32")
    vocab = shape[-1]
    n = logits.numel() // vocab if vocab else 0
    if temperature is not None and (temperature.dtype is not _F32 or temperature.shape != shape[:-1]
                                    or not temperature.is_contiguous()):
        raise ValueError("temperature: f32, one a row")
    dev, stream = _place(logits, temperature, out)
    if out is None:
        out = torch.empty_like(logits)
    elif out.shape != shape or out.dtype is not _F32 or not out.is_contiguous():
        raise ValueError("out: as logits")
    nb = _probs_ws(n, vocab)
    ws = torch.empty(nb, dtype=_U8, device=dev) if nb else None
    rc = lib().loomhip_token_probs_dev(logits.data_ptr(), n, vocab, vocab,
                                       None if temperature is None else temperature.data_ptr(), out.data_ptr(), vocab,
                                       ws.data_ptr() if nb else None, nb, stream)
    if rc != OK:
        _fail("token_probs_dev", rc)
    return out


def _is(t, dtype, *shape) -> bool:
    return t.shape == shape and t.dtype is dtype and t.is_contiguous()


def verify_drafts_dev(target_probs, draft_tokens, u_accept, u_sample, draft_probs=None, n_draft=None):
    """Drafted tokens against the target's probabilities, from given random numbers in [0, 1).

    target_probs f32 [n, k + 1, vocab], draft_tokens int32 [n, k], u_accept f32 [n, k], u_sample f32 [n], draft_probs
    f32 [n, k, vocab] (None: a drafter that names one token), n_draft int32 [n] (None: k each).  Returns (tokens int32
    [n, k + 1]: the accepted ones, the next one, then -1; accepted int32 [n]).
    """
    if target_probs.dim() != 3 or target_probs.shape[1] < 1:
        raise ValueError("target_probs: f32 [n, k + 1, vocab]")
    n, k1, vocab = target_probs.shape
    k = k1 - 1
    if not (_is(target_probs, _F32, n, k1, vocab) and _is(draft_tokens, _I32, n, k) and _is(u_accept, _F32, n, k)
            and _is(u_sample, _F32, n) and (draft_probs is None or _is(draft_probs, _F32, n, k, vocab))
            and (n_draft is None or _is(n_draft, _I32, n))):
        raise ValueError(f"contiguous target_probs f32 [{n}, {k1}, {vocab}], draft_tokens int32 [{n}, {k}], u_accept f32 "
                         f"[{n}, {k}], u_sample f32 [{n}], draft_probs f32 [{n}, {k}, {vocab}], n_draft int32 [{n}]")
    dev, stream = _place(target_probs, draft_tokens, u_accept, u_sample, draft_probs, n_draft)
    tokens = torch.empty((n, k1), dtype=_I32, device=dev)
    accepted = torch.empty((n,), dtype=_I32, device=dev)
    nb = _verify_ws(n, vocab)
    ws = torch.empty(nb, dtype=_U8, device=dev) if nb else None
    rc = lib().loomhip_verify_drafts_dev(
        target_probs.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(), draft_tokens.data_ptr(),
        None if n_draft is None else n_draft.data_ptr(), u_accept.data_ptr(), u_sample.data_ptr(), n, k, vocab,
        tokens.data_ptr(), accepted.data_ptr(), ws.data_ptr() if nb else None, nb, stream)
    if rc != OK:
        _fail("verify_drafts_dev", rc)
    return tokens, accepted


__all__ = ["lora_dev", "prefix_attn_dev", "token_probs_dev", "verify_drafts_dev"]
