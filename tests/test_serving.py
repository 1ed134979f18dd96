"""The batched serving operators without a GPU: what they refuse before
anything could be launched, and their workspaces."""
import ctypes as C

import pytest
import torch

import loom_amd
from loom_amd import serving

FAKE = 0x1000  # an address for checks that come before any access


def _attn(prefix=None, own=None, q=FAKE, own_len=FAKE, q_len=None, n=2, n_q=1, heads=4, kv=2, hd=64, out=FAKE, ws=FAKE,
          ws_bytes=1 << 40):
    L = loom_amd.lib()
    pre = loom_amd.KvRowsDesc(*(prefix or (FAKE, FAKE, 16, 0, 128, 64)))
    mine = loom_amd.KvRowsDesc(*(own or (FAKE, FAKE, 8, 1024, 128, 64)))
    return L.loomhip_prefix_attn_dev(C.byref(pre), C.byref(mine), q, own_len, q_len, n, n_q, heads, kv, hd, 0.125, out, 0, ws,
                                     ws_bytes, None)


@pytest.mark.parametrize("rc,args", [
    (loom_amd.ERR_ARG, dict(q=None)),
    (loom_amd.ERR_ARG, dict(out=None)),
    (loom_amd.ERR_ARG, dict(own_len=None)),
    (loom_amd.ERR_ARG, dict(heads=5)),
    (loom_amd.ERR_ARG, dict(kv=0)),
    (loom_amd.ERR_ARG, dict(prefix=(None, FAKE, 16, 0, 128, 64))),
    (loom_amd.ERR_ARG, dict(own=(FAKE, None, 8, 1024, 128, 64))),
    (loom_amd.ERR_ARG, dict(own=(FAKE, FAKE, 8, 1024, 32, 64))),
    (loom_amd.DECLINED, dict(hd=0)),
    (loom_amd.DECLINED, dict(hd=60)),
    (loom_amd.DECLINED, dict(hd=264)),
    (loom_amd.DECLINED, dict(q=FAKE + 4)),
    (loom_amd.DECLINED, dict(out=FAKE + 8)),
    (loom_amd.DECLINED, dict(prefix=(FAKE + 2, FAKE, 16, 0, 128, 64))),
    (loom_amd.DECLINED, dict(prefix=(FAKE, FAKE, 16, 0, 132, 64))),
    (loom_amd.DECLINED, dict(own=(FAKE, FAKE, 8, 1028, 128, 64))),
    (loom_amd.DECLINED, dict(own=(FAKE, FAKE, 8, 1024, 128, 68))),
    (loom_amd.DECLINED, dict(prefix=(FAKE, FAKE, 1 << 40, 0, 128, 64))),
    (loom_amd.DECLINED, dict(n=1 << 20)),
    (loom_amd.DECLINED, dict(n_q=1 << 20)),
    (loom_amd.ERR_ARG, dict(ws=None)),
    (loom_amd.ERR_ARG, dict(ws=FAKE + 8)),
    (loom_amd.ERR_ARG, dict(ws_bytes=2 * 4 * (64 * 4 + 8))),
    (loom_amd.DECLINED, dict(prefix=(FAKE, FAKE, 16, 0, 1 << 24, 64))),
    (loom_amd.DECLINED, dict(own=(FAKE, FAKE, 8, 1 << 30, 1 << 24, 64))),
])
def test_prefix_attn_refuses(rc, args):
    assert _attn(**args) == rc
    assert "prefix_attn" in loom_amd.last_error()


def test_nothing_to_do_is_ok():
    L = loom_amd.lib()
    assert _attn(n=0) == loom_amd.OK and _attn(n_q=0) == loom_amd.OK
    d = loom_amd.LoraDesc(loom_amd.F16, 1, 8, 64, 64, FAKE, FAKE, FAKE)
    assert L.loomhip_lora_dev(C.byref(d), None, 64, None, None, 64, 0, None, 64, None, 0, None) == loom_amd.OK
    assert L.loomhip_token_probs_dev(None, 0, 64, 64, None, None, 64, None, 0, None) == loom_amd.OK
    assert L.loomhip_verify_drafts_dev(None, None, None, None, None, None, 0, 4, 64, None, None, None, 0, None) == loom_amd.OK


def _lora(type=loom_amd.F16, adapters=2, rank=8, rows=64, cols=32, a=FAKE, b=FAKE, scale=FAKE, x=0x100000, xs=32, ids=FAKE,
          base=None, bs=64, n=4, out=0x200000, os=64, ws=FAKE, ws_bytes=1 << 40):
    d = loom_amd.LoraDesc(type, adapters, rank, rows, cols, a, b, scale)
    return loom_amd.lib().loomhip_lora_dev(C.byref(d), x, xs, ids, base, bs, n, out, os, ws, ws_bytes, None)


@pytest.mark.parametrize("rc,args", [
    (loom_amd.DECLINED, dict(type=loom_amd.Q4_0)),
    (loom_amd.DECLINED, dict(rank=0)),
    (loom_amd.DECLINED, dict(rank=257)),
    (loom_amd.ERR_ARG, dict(adapters=0)),
    (loom_amd.ERR_ARG, dict(rows=0)),
    (loom_amd.ERR_ARG, dict(cols=0)),
    (loom_amd.ERR_ARG, dict(a=None)),
    (loom_amd.ERR_ARG, dict(scale=None)),
    (loom_amd.ERR_ARG, dict(x=None)),
    (loom_amd.ERR_ARG, dict(ids=None)),
    (loom_amd.ERR_ARG, dict(out=None)),
    (loom_amd.ERR_ARG, dict(xs=31)),
    (loom_amd.ERR_ARG, dict(os=63)),
    (loom_amd.ERR_ARG, dict(base=0x300000, bs=63)),
    (loom_amd.ERR_ARG, dict(a=FAKE + 1)),
    (loom_amd.ERR_ARG, dict(x=0x100002)),
    (loom_amd.ERR_ARG, dict(rank=128, ws=None)),
    (loom_amd.ERR_ARG, dict(rank=128, ws=FAKE + 8)),
    (loom_amd.ERR_ARG, dict(rank=128, ws_bytes=255)),
    (loom_amd.DECLINED, dict(n=65535 * 64 + 1)),
    (loom_amd.ERR_ARG, dict(out=0x100000)),               # over x
    (loom_amd.ERR_ARG, dict(out=0x100000 - 4)),           # into x
    (loom_amd.ERR_ARG, dict(base=0x200004)),              # over base, shifted
    (loom_amd.ERR_ARG, dict(base=0x200000, bs=128)),      # base's rows elsewhere than out's
])
def test_lora_refuses(rc, args):
    assert _lora(**args) == rc
    assert "lora" in loom_amd.last_error()


@pytest.mark.parametrize("rc,args", [
    (loom_amd.ERR_ARG, dict(logits=None)),
    (loom_amd.ERR_ARG, dict(probs=None)),
    (loom_amd.ERR_ARG, dict(vocab=0)),
    (loom_amd.ERR_ARG, dict(stride=99)),
    (loom_amd.ERR_ARG, dict(os=99)),
    (loom_amd.ERR_ARG, dict(logits=FAKE + 2)),
    (loom_amd.ERR_ARG, dict(t=FAKE + 1)),
    (loom_amd.ERR_ARG, dict(probs=0x100002)),
    (loom_amd.ERR_ARG, dict(vocab=40000, stride=40000, os=40000, ws=None)),
    (loom_amd.ERR_ARG, dict(vocab=40000, stride=40000, os=40000, ws=FAKE + 8)),
    (loom_amd.ERR_ARG, dict(vocab=40000, stride=40000, os=40000, ws_bytes=15)),
    (loom_amd.DECLINED, dict(n=65536)),
    (loom_amd.DECLINED, dict(vocab=1 << 31, stride=1 << 31, os=1 << 31)),
])
def test_token_probs_refuses(rc, args):
    a = dict(logits=FAKE, n=3, vocab=100, stride=100, t=None, probs=0x100000, os=100, ws=FAKE, ws_bytes=1 << 40) | args
    L = loom_amd.lib()
    assert L.loomhip_token_probs_dev(a["logits"], a["n"], a["vocab"], a["stride"], a["t"], a["probs"], a["os"], a["ws"],
                                     a["ws_bytes"], None) == rc
    assert "token_probs" in loom_amd.last_error()


@pytest.mark.parametrize("rc,args", [
    (loom_amd.ERR_ARG, dict(target=None)),
    (loom_amd.ERR_ARG, dict(tok=None)),
    (loom_amd.ERR_ARG, dict(ua=None)),
    (loom_amd.ERR_ARG, dict(us=None)),
    (loom_amd.ERR_ARG, dict(out=None)),
    (loom_amd.ERR_ARG, dict(acc=None)),
    (loom_amd.ERR_ARG, dict(target=FAKE + 2)),
    (loom_amd.ERR_ARG, dict(us=FAKE + 1)),
    (loom_amd.ERR_ARG, dict(out=FAKE + 2)),
    (loom_amd.ERR_ARG, dict(vocab=0)),
    (loom_amd.ERR_ARG, dict(vocab=40000, ws=None)),
    (loom_amd.ERR_ARG, dict(vocab=40000, ws=FAKE + 4)),
    (loom_amd.ERR_ARG, dict(vocab=40000, ws_bytes=8)),
    (loom_amd.DECLINED, dict(n=65536)),
    (loom_amd.DECLINED, dict(k=4097)),
    (loom_amd.DECLINED, dict(vocab=1 << 31)),
])
def test_verify_drafts_refuses(rc, args):
    a = dict(target=FAKE, draft=FAKE, tok=FAKE, nd=None, ua=FAKE, us=FAKE, n=3, k=2, vocab=100, out=FAKE, acc=FAKE, ws=FAKE,
             ws_bytes=1 << 40) | args
    L = loom_amd.lib()
    assert L.loomhip_verify_drafts_dev(a["target"], a["draft"], a["tok"], a["nd"], a["ua"], a["us"], a["n"], a["k"],
                                       a["vocab"], a["out"], a["acc"], a["ws"], a["ws_bytes"], None) == rc
    assert "verify_drafts" in loom_amd.last_error()


def test_without_a_device_the_calls_say_so():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert _attn() == loom_amd.ERR_INIT
    assert _lora() == loom_amd.ERR_INIT


def test_workspaces_grow_with_the_call():
    L = loom_amd.lib()
    assert L.loomhip_token_probs_ws(0, 100) == 0 and L.loomhip_verify_drafts_ws(0, 100) == 0
    assert L.loomhip_token_probs_ws(5, 0) == 0 and L.loomhip_verify_drafts_ws(5, 0) == 0
    d = loom_amd.LoraDesc(loom_amd.F16, 1, 8, 64, 64, FAKE, FAKE, FAKE)
    assert L.loomhip_lora_ws(C.byref(d), 0) == 0 and L.loomhip_lora_ws(None, 4) == 0
    assert L.loomhip_lora_ws(C.byref(d), 1) == 0  # one launch
    d = loom_amd.LoraDesc(loom_amd.F16, 1, 128, 64, 64, FAKE, FAKE, FAKE)
    assert 0 < L.loomhip_lora_ws(C.byref(d), 1) <= L.loomhip_lora_ws(C.byref(d), 1000)
    for bad in (loom_amd.LoraDesc(loom_amd.F16, 1, 0, 64, 64), loom_amd.LoraDesc(loom_amd.F16, 1, 8, 0, 64),
                loom_amd.LoraDesc(loom_amd.F16, 1, 8, 64, 0), loom_amd.LoraDesc(loom_amd.F16, 1, 257, 64, 64)):
        assert L.loomhip_lora_ws(C.byref(bad), 4) == 0
    assert L.loomhip_prefix_attn_ws(100, 10, 0, 1, 8, 2, 64) == 0
    assert L.loomhip_prefix_attn_ws(100, 10, 2, 0, 8, 2, 64) == 0
    assert L.loomhip_prefix_attn_ws(100, 10, 2, 1, 8, 0, 64) == 0
    assert L.loomhip_prefix_attn_ws(0, 0, 2, 1, 8, 2, 64) == 0
    assert L.loomhip_prefix_attn_ws(100, 10, 2, 1, 8, 2, 64) >= 2 * 8 * 64 * 4 * 2
    for n, vocab in ((1, 1), (1, 8192), (65535, 7)):  # one launch
        assert L.loomhip_token_probs_ws(n, vocab) == 0
        assert L.loomhip_verify_drafts_ws(n, vocab) == 0
    for n, vocab in ((1, 32769), (64, 151936), (65535, 50257)):
        assert L.loomhip_token_probs_ws(n, vocab) >= 16 * n
        assert L.loomhip_verify_drafts_ws(n, vocab) >= 16 * n


def _bad(call, *a, **k):
    with pytest.raises(ValueError):
        call(*a, **k)


def test_python_entry_points_refuse_wrong_tensors():
    f, h, i = torch.float32, torch.float16, torch.int32
    q, kp, ko = torch.zeros(2, 1, 4, 64), torch.zeros(8, 2, 64, dtype=h), torch.zeros(2, 8, 2, 64, dtype=h)
    ln = torch.ones(2, dtype=i)
    _bad(serving.prefix_attn_dev, q.half(), kp, kp, ko, ko, ln, 1.0)
    _bad(serving.prefix_attn_dev, q.transpose(1, 2), kp, kp, ko, ko, ln, 1.0)
    _bad(serving.prefix_attn_dev, q, kp.float(), kp.float(), ko, ko, ln, 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp[:4], ko, ko, ln, 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp, ko[:1], ko[:1], ln, 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp, ko[..., :1, :], ko[..., :1, :], ln, 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp, ko, ko, None, 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp, ko, ko, ln.long(), 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp, ko, ko, ln, 1.0, q_len=torch.ones(3, dtype=i))
    _bad(serving.prefix_attn_dev, q, None, None, None, None, None, 1.0)
    _bad(serving.prefix_attn_dev, q, kp, kp, ko, ko, ln, 1.0, out=torch.zeros(2, 1, 4, 32))
    _bad(serving.prefix_attn_dev, q, kp, kp, ko, ko, ln, 1.0)  # everything right but the device
    x, a, b = torch.zeros(3, 32), torch.zeros(2, 4, 32, dtype=h), torch.zeros(2, 16, 4, dtype=h)
    sc, ids = torch.zeros(2), torch.zeros(3, dtype=i)
    _bad(serving.lora_dev, x.half(), a, b, sc, ids)
    _bad(serving.lora_dev, x, a, b.float(), sc, ids)
    _bad(serving.lora_dev, x, a.to(torch.int8), b.to(torch.int8), sc, ids)
    _bad(serving.lora_dev, x, a, b[:, :, :3], sc, ids)
    _bad(serving.lora_dev, x, a, b, sc[:1], ids)
    _bad(serving.lora_dev, x, a, b, sc, ids.long())
    _bad(serving.lora_dev, x, a, b, sc, ids, base=torch.zeros(3, 15))
    _bad(serving.lora_dev, x, a, b, sc, ids, out=torch.zeros(16, 3).t())
    _bad(serving.lora_dev, x, a, b, sc, ids, out=torch.zeros(1, 16).expand(3, 16))
    _bad(serving.lora_dev, x, a, b, sc, ids)
    _bad(serving.token_probs_dev, torch.zeros(2, 8, dtype=torch.float64))
    _bad(serving.token_probs_dev, torch.zeros(8, 2).t())
    _bad(serving.token_probs_dev, torch.zeros(2, 8), torch.zeros(3))
    _bad(serving.token_probs_dev, torch.zeros(2, 8), out=torch.zeros(2, 9))
    _bad(serving.token_probs_dev, torch.zeros(2, 8))
    t, d = torch.zeros(2, 4, 9), torch.zeros(2, 3, 9)
    tok, ua, us = torch.zeros(2, 3, dtype=i), torch.zeros(2, 3), torch.zeros(2)
    _bad(serving.verify_drafts_dev, t[0], tok, ua, us)
    _bad(serving.verify_drafts_dev, t, tok.long(), ua, us)
    _bad(serving.verify_drafts_dev, t, tok, ua[:, :2], us)
    _bad(serving.verify_drafts_dev, t, tok, ua, us[:1])
    _bad(serving.verify_drafts_dev, t, tok, ua, us, draft_probs=d[:, :2])
    _bad(serving.verify_drafts_dev, t, tok, ua, us, draft_probs=d, n_draft=torch.zeros(3, dtype=i))
    _bad(serving.verify_drafts_dev, t, tok, ua, us, draft_probs=d)
