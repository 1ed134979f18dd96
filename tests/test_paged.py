"""The operators around a paged cache without a GPU: what they refuse before
anything could be launched, their workspaces, and the definitions they are
tested against."""
import ctypes as C

import numpy as np
import pytest
import torch

import loom_amd
import paged_ref as ref
from loom_amd import serving

FAKE = 0x1000  # an address for checks that come before any access
F16, BF16, OK, ARG, DECLINED = loom_amd.F16, loom_amd.BF16, loom_amd.OK, loom_amd.ERR_ARG, loom_amd.DECLINED


def _pages(k=FAKE, v=FAKE, type=F16, n_pages=8, page_size=16, page_stride=2048, row_stride=128, head_stride=64, table=FAKE,
           n_lanes=4, table_width=4, table_stride=4):
    return loom_amd.PagesDesc(k, v, type, n_pages, page_size, page_stride, row_stride, head_stride, table, n_lanes,
                              table_width, table_stride)


def _rope(n=4, hd=64, q=None, k=None, pos=FAKE, freqs=FAKE, rot=64):
    qd = loom_amd.HeadsDesc(*(q or (0x100000, 256, 0x200000, 256, None, 4)))
    kd = loom_amd.HeadsDesc(*(k or (0x300000, 128, 0x400000, 128, None, 2)))
    r = loom_amd.RopeDesc(pos, freqs, rot, 0, 1e-6)
    return loom_amd.lib().loomhip_qk_norm_rope_dev(C.byref(qd), C.byref(kd), C.byref(r), n, hd, None)


@pytest.mark.parametrize("rc,args", [
    (ARG, dict(pos=None)),
    (ARG, dict(freqs=None)),
    (ARG, dict(rot=63)),
    (ARG, dict(rot=66)),
    (ARG, dict(pos=FAKE + 2)),
    (ARG, dict(freqs=FAKE + 4)),
    (DECLINED, dict(hd=0, rot=0)),
    (DECLINED, dict(hd=60, rot=0)),
    (DECLINED, dict(hd=264)),
    (DECLINED, dict(n=(1 << 23) + 1)),
    (ARG, dict(q=(None, 256, 0x200000, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, None, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, 0x200000, 256, None, 0))),
    (ARG, dict(q=(0x100000, 255, 0x200000, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, 0x200000, 255, None, 4))),
    (ARG, dict(q=(0x100002, 256, 0x200000, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, 0x200000, 256, 0x501, 4))),
    (DECLINED, dict(q=(0x100000, 1 << 20, 0x90000000, 1 << 20, None, 5000))),
    (ARG, dict(k=(None, 128, 0x400000, 128, None, 2))),
    (ARG, dict(k=(0x300000, 128, None, 128, None, 2))),
    # an output over the other input, the other output, or its own input without being it
    (ARG, dict(q=(0x100000, 256, 0x300000, 256, None, 4))),
    (ARG, dict(k=(0x300000, 128, 0x100000, 128, None, 2))),
    (ARG, dict(k=(0x300000, 128, 0x200100, 128, None, 2))),
    (ARG, dict(q=(0x100000, 256, 0x100100, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, 0x100000, 512, None, 4))),
])
def test_qk_norm_rope_refuses(rc, args):
    assert _rope(**args) == rc
    assert "qk_norm_rope" in loom_amd.last_error()


def _append(pages=None, n=4, hd=64, q=(0x100000, 256, 0x200000, 256, None, 4), k=(0x300000, 128, None, 0, None, 2),
            v=0x400000, vs=128, lanes=None, pos=FAKE, freqs=FAKE, rot=64):
    qd = C.byref(loom_amd.HeadsDesc(*q)) if q else None
    r = loom_amd.RopeDesc(pos, freqs, rot, 0, 1e-6)
    return loom_amd.lib().loomhip_paged_append_dev(C.byref(pages or _pages()), qd, C.byref(loom_amd.HeadsDesc(*k)), v, vs,
                                                   lanes, C.byref(r), n, hd, None)


BAD_PAGES = [
    (ARG, dict(k=None)),
    (ARG, dict(v=None)),
    (ARG, dict(table=None)),
    (ARG, dict(table=FAKE + 2)),
    (DECLINED, dict(type=loom_amd.F32)),
    (DECLINED, dict(type=loom_amd.Q8_0)),
    (ARG, dict(n_pages=0)),
    (ARG, dict(page_size=0)),
    (ARG, dict(n_lanes=0)),
    (ARG, dict(table_width=0)),
    (ARG, dict(table_stride=3)),
    (DECLINED, dict(n_pages=1 << 31)),
    (DECLINED, dict(page_size=1 << 31)),
    (DECLINED, dict(table_width=1 << 28, table_stride=1 << 28)),
    (DECLINED, dict(page_stride=1 << 33)),
    (DECLINED, dict(row_stride=1 << 33)),
    (DECLINED, dict(n_pages=1 << 30)),
    (DECLINED, dict(page_stride=2044)),
    (DECLINED, dict(row_stride=132)),
    (DECLINED, dict(head_stride=68)),
    (DECLINED, dict(k=FAKE + 8)),
    (DECLINED, dict(v=FAKE + 2)),
    (ARG, dict(row_stride=0)),
    (ARG, dict(head_stride=32)),
    (ARG, dict(page_stride=0)),
]


@pytest.mark.parametrize("rc,args", BAD_PAGES)
def test_pages_are_refused(rc, args):
    assert _append(pages=_pages(**args)) == rc
    assert "paged_append" in loom_amd.last_error()
    assert _attn(pages=_pages(**args)) == rc
    assert "paged_attn" in loom_amd.last_error()


@pytest.mark.parametrize("rc,args", [
    (ARG, dict(pos=None)),
    (ARG, dict(rot=2, freqs=None)),
    (ARG, dict(v=None)),
    (ARG, dict(k=(None, 128, None, 0, None, 2))),
    (ARG, dict(k=(0x300000, 128, None, 0, None, 0))),
    (ARG, dict(k=(0x300000, 127, None, 0, None, 2))),
    (ARG, dict(vs=127)),
    (ARG, dict(v=0x400001)),
    (ARG, dict(lanes=FAKE + 1)),
    (ARG, dict(n=5)),
    (ARG, dict(q=(0x100000, 256, None, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, 0x300000, 256, None, 4))),
    (ARG, dict(q=(0x100000, 256, 0x400000, 256, None, 4))),
    (DECLINED, dict(hd=72, rot=0, k=(0x300000, 1 << 33, None, 0, None, 2))),
])
def test_paged_append_refuses(rc, args):
    assert _append(**args) == rc
    assert "paged_append" in loom_amd.last_error()


def test_paged_append_refuses_one_pool_for_keys_and_values():
    """Their rows would be written by two threads each."""
    assert _append(pages=_pages(k=0x600000, v=0x600000)) == ARG
    assert "one pool" in loom_amd.last_error()


def _attn(pages=None, q=FAKE, lens=FAKE, n=2, heads=4, kv=2, hd=64, window=0, out=FAKE, ws=FAKE, ws_bytes=1 << 40):
    return loom_amd.lib().loomhip_paged_attn_dev(C.byref(pages or _pages()), q, lens, n, heads, kv, hd, 0.125, window, out, ws,
                                                 ws_bytes, None)


@pytest.mark.parametrize("rc,args", [
    (ARG, dict(q=None)),
    (ARG, dict(out=None)),
    (ARG, dict(lens=None)),
    (ARG, dict(lens=FAKE + 2)),
    (ARG, dict(heads=5)),
    (ARG, dict(kv=0)),
    (ARG, dict(n=5)),
    (DECLINED, dict(hd=0)),
    (DECLINED, dict(hd=60)),
    (DECLINED, dict(hd=264)),
    (DECLINED, dict(n=1 << 20)),
    (DECLINED, dict(n=1 << 15, heads=(1 << 8) + 2, pages=_pages(n_lanes=1 << 15))),
    (DECLINED, dict(q=FAKE + 4)),
    (DECLINED, dict(out=FAKE + 8)),
    (ARG, dict(pages=_pages(page_size=256, page_stride=32768), ws=None)),
    (ARG, dict(pages=_pages(page_size=256, page_stride=32768), ws=FAKE + 8)),
    (ARG, dict(pages=_pages(page_size=256, page_stride=32768), ws_bytes=4096)),
    (DECLINED, dict(pages=_pages(table_width=1 << 26, table_stride=1 << 26, n_lanes=1 << 9), n=1 << 9)),
])
def test_paged_attn_refuses(rc, args):
    assert _attn(**args) == rc
    assert "paged_attn" in loom_amd.last_error()


def _logprobs(logits=FAKE, n=4, vocab=1000, stride=1000, tokens=FAKE, temperature=None, top=3, lp=FAKE, entropy=FAKE,
              ids=FAKE, tops=FAKE, ws=FAKE, ws_bytes=1 << 40):
    return loom_amd.lib().loomhip_token_logprobs_dev(logits, n, vocab, stride, tokens, temperature, top, lp, entropy, ids, tops,
                                                     ws, ws_bytes, None)


@pytest.mark.parametrize("rc,args", [
    (ARG, dict(logits=None)),
    (ARG, dict(tokens=None)),
    (ARG, dict(lp=None)),
    (ARG, dict(entropy=None)),
    (ARG, dict(ids=None)),
    (ARG, dict(tops=None)),
    (ARG, dict(vocab=0)),
    (ARG, dict(stride=999)),
    (ARG, dict(logits=FAKE + 2)),
    (ARG, dict(temperature=FAKE + 1)),
    (ARG, dict(ids=FAKE + 2)),
    (DECLINED, dict(top=33)),
    (DECLINED, dict(n=65536)),
    (DECLINED, dict(vocab=(1 << 21) + 1, stride=1 << 22)),
    (ARG, dict(vocab=151936, stride=151936, ws=None)),
    (ARG, dict(vocab=151936, stride=151936, ws=FAKE + 8)),
    (ARG, dict(vocab=151936, stride=151936, ws_bytes=64)),
])
def test_token_logprobs_refuses(rc, args):
    assert _logprobs(**args) == rc
    assert "token_logprobs" in loom_amd.last_error()


def test_nothing_to_do_is_ok():
    L = loom_amd.lib()
    assert _rope(n=0) == OK and _append(n=0) == OK and _attn(n=0) == OK and _logprobs(n=0) == OK
    assert L.loomhip_token_logprobs_ws(0, 151936, 20) == 0 and L.loomhip_paged_attn_ws(4096, 0, 32, 4, 128) == 0


def test_attn_workspace():
    """None where no lane is cut; else room for the records of every cut that the lengths can lead to."""
    ws = loom_amd.lib().loomhip_paged_attn_ws
    assert ws(512, 64, 32, 4, 128) == 0 and ws(256, 64, 32, 4, 256) == 0
    for rows, n, heads, kv, hd in ((513, 1, 32, 4, 128), (1 << 20, 64, 32, 4, 128), (1 << 20, 65535, 32, 32, 64), (300, 9, 40, 1, 256)):
        items = n * kv * -(-(heads // kv) // 16)
        room = 256 if hd > 128 else 512
        records, cols = room * (1 if items <= room // 2 else 4), min(heads // kv, 16)
        assert ws(rows, n, heads, kv, hd) == 16 + records * (8 + cols * (hd * 4 + 8))
        # the plan's own bounds, over lengths drawn at random: lanes of u units in pieces of at most L
        r = np.random.default_rng(rows)
        for spread in (1, 30, 3000):
            u = r.integers(0, spread + 1, min(n, 3000))
            it = items // n
            share = -(-int(u.sum()) * it // room)
            pieces = lambda L: np.maximum(1, -(-u // L))
            cuts = [max(1, -(-share * s // 16)) for s in (16, 17, 18, 20, 24, 32)]
            L = next((c for c in cuts if pieces(c).sum() * it <= room), max(1, (share + 1) // 2))
            p = pieces(L)
            assert p[p > 1].sum() * it <= 4 * room
            if len(u) * it <= room // 2:
                assert p.sum() * it <= room


def test_logprobs_workspace():
    L = loom_amd.lib()
    assert L.loomhip_token_logprobs_ws(5, 32000, 32) == 0  # a work group holds the row
    for n, vocab, top in ((1, 151936, 0), (1, 151936, 32), (64, 151936, 20), (65535, 40000, 1), (1, 1 << 21, 32)):
        nb = L.loomhip_token_logprobs_ws(n, vocab, top)
        parts = nb // (n * (16 + 8 * top))
        assert nb == n * parts * (16 + 8 * top) and parts * 2048 * 8 >= vocab and parts * max(top, 1) <= 4096


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_python_checks():
    """Wrong tensors raise ValueError before anything else; the right ones fail only at the device."""
    i32 = torch.int32
    f = _t(32, dtype=torch.float64)
    q, k, v = _t(3, 4, 64), _t(3, 2, 64), _t(3, 2, 64)
    kp, vp, table, pos = _t(5, 16, 2, 64, dtype=torch.float16), _t(5, 16, 2, 64, dtype=torch.float16), _t(3, 4, dtype=i32), _t(3, dtype=i32)
    good = [lambda **x: serving.qk_norm_rope_dev(**{**dict(q=q, k=k, pos=pos, freqs=f), **x}),
            lambda **x: serving.paged_append_dev(**{**dict(k=k, v=v, k_pages=kp, v_pages=vp, table=table, pos=pos, freqs=f), **x}),
            lambda **x: serving.paged_attn_dev(**{**dict(q=q, k_pages=kp, v_pages=vp, table=table, lens=pos, scale=0.1), **x}),
            lambda **x: serving.token_logprobs_dev(**{**dict(logits=_t(3, 100), tokens=pos, top=2), **x})]
    wrong = [
        [dict(q=_t(3, 256)), dict(q=q.half()), dict(pos=pos.long()), dict(pos=_t(2, dtype=i32)), dict(freqs=f.float()),
         dict(freqs=_t(2, 3, dtype=torch.float64)), dict(q_norm=_t(63)), dict(k_norm=_t(64).half()), dict(k=_t(3, 2, 32)),
         dict(k=None, k_out=k), dict(q_out=_t(3, 4, 32)), dict(k=_t(2, 2, 64)), dict(q=_t(3, 64, 4).transpose(1, 2))],
        [dict(v=_t(3, 2, 32)), dict(k=k.half()), dict(lanes=_t(3)), dict(lanes=_t(2, dtype=i32)), dict(table=_t(3, 4)),
         dict(table=_t(12, dtype=i32)), dict(table=_t(4, 3, dtype=i32).t()), dict(k_pages=kp.float(), v_pages=vp.float()),
         dict(v_pages=vp.bfloat16()), dict(k_pages=_t(5, 16, 4, 64, dtype=torch.float16)), dict(v_pages=vp[:4]),
         dict(k_pages=kp.transpose(1, 2).contiguous().transpose(1, 2)), dict(q_out=q), dict(q=_t(3, 4, 32)), dict(q_norm=_t(3))],
        [dict(q=q.double()), dict(q=_t(3, 4, 65)), dict(lens=_t(2, dtype=i32)), dict(lens=_t(3)), dict(window=-1),
         dict(out=_t(3, 4, 32)), dict(k_pages=kp[0], v_pages=vp[0]), dict(q=_t(3, 4, 128)[..., ::2])],
        [dict(logits=_t(3, 100).half()), dict(logits=_t(100, 3).t()), dict(tokens=pos.long()), dict(tokens=_t(4, dtype=i32)),
         dict(temperature=_t(4)), dict(top=-1)],
    ]
    for call, cases in zip(good, wrong):
        with pytest.raises(ValueError, match="not on the GPU"):
            call()
        for x in cases:
            with pytest.raises(ValueError) as e:
                call(**x)
            assert "on the GPU" not in str(e.value), x


def test_log_probabilities_of_no_vocabulary_are_refused():
    """Rows without values have no results that could be left unwritten; no rows are nothing to do, whatever their length."""
    for shape in ((3, 0), (2, 3, 0), (0,)):
        with pytest.raises(ValueError, match="no values"):
            serving.token_logprobs_dev(_t(*shape), _t(*shape[:-1], dtype=torch.int32), top=2)
    with pytest.raises(ValueError, match="not on the GPU"):
        serving.token_logprobs_dev(_t(0, 0), _t(0, dtype=torch.int32), top=2)


def test_rotation_keeps_lengths_and_relative_angles():
    """The definition: rotated pairs keep their length, and (q at p) . (k at r) hangs on p - r alone."""
    r = np.random.default_rng(1)
    x, y = r.standard_normal((1, 1, 32)), r.standard_normal((1, 1, 32))
    freqs = 1.0 / 10000.0 ** (np.arange(0, 32, 2) / 32)
    for inter in (False, True):
        turn = lambda a, p: ref.norm_rope(a, [p], freqs, None, 0, inter)[0][0, 0]
        assert abs(np.linalg.norm(turn(x, 917)) - np.linalg.norm(x)) < 1e-12
        assert abs(turn(x, 917) @ turn(y, 900) - turn(x, 17) @ turn(y, 0)) < 1e-9
        assert abs(turn(x, 17) @ turn(y, 0) - turn(x, 18) @ turn(y, 0)) > 1e-3
