"""What the batched serving operators take and refuse by where their tensors
lie, without a GPU: a call that passes its checks ends at the missing device."""
import ctypes as C

import pytest
import torch

import loom_amd

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: a GPU would be given them")

FAKE = 0x1000
PASSED = loom_amd.ERR_INIT


def _lora(x, xs, base, bs, out, os, n=4, rows=64, cols=32):
    d = loom_amd.LoraDesc(loom_amd.F16, 2, 8, rows, cols, FAKE, FAKE, FAKE)
    return loom_amd.lib().loomhip_lora_dev(C.byref(d), x, xs, FAKE, base, bs, n, out, os, FAKE, 1 << 40, None)


AT = 0x100000  # a buffer


def _takes(x, xs, base, bs, out, os, n, rows, cols):
    """The definition: the elements of out's rows, and of x's and base's."""
    def elements(p, s, w):
        return {p + 4 * (i * s + c) for i in range(n) for c in range(w)}

    o = elements(out, os, rows)
    same = base == out and bs == os
    return not (o & elements(x, xs, cols)) and (base is None or same or not (o & elements(base, bs, rows)))


def test_lora_column_groups_of_one_buffer():
    """Every placement of out against x and base in rows of 24 values: taken exactly where no element is shared."""
    n, rows, cols, s = 3, 5, 4, 24
    taken = 0
    for d in range(-3 * s - 8, 3 * s + 9):  # out's first element from x's
        out = AT + 4 * d
        for base in (None, out, AT + 4 * 10, AT + 4 * (s + 10)):
            want = _takes(AT, s, base, s, out, s, n, rows, cols)
            taken += want
            assert _lora(AT, s, base, s, out, s, n, rows, cols) == (PASSED if want else loom_amd.ERR_ARG), (d, base)
    assert taken > 100
    assert _lora(AT, 4, AT + 400, 5, AT + 400, 9, 1, 5, 4) == PASSED  # in place, one row: its stride has no part in it
    for d in range(-8, 9):  # rows one after the other, and a single row
        for n, s in ((3, 5), (1, 5), (1, 1000)):
            out = AT + 4 * d
            want = _takes(AT, s, None, s, out, s, n, 5, 4)
            assert _lora(AT, s, None, s, out, s, n, 5, 4) == (PASSED if want else loom_amd.ERR_ARG), (d, n, s)


def _probs(logits, stride, probs, os, n=3, vocab=5):
    return loom_amd.lib().loomhip_token_probs_dev(logits, n, vocab, stride, None, probs, os, FAKE, 1 << 40, None)


def test_token_probs_over_its_logits():
    """In place with the same rows, or rows that share no element."""
    for s in (5, 11, 24):
        logits = {AT + 4 * (i * s + c) for i in range(3) for c in range(5)}
        for d in range(-3 * s - 8, 3 * s + 9):
            want = d == 0 or not logits & {a + 4 * d for a in logits}
            assert _probs(AT, s, AT + 4 * d, s) == (PASSED if want else loom_amd.ERR_ARG), (s, d)
    for s, os in ((5, 6), (6, 5), (24, 5)):  # the same first element, other rows
        assert _probs(AT, s, AT, os) == loom_amd.ERR_ARG
        assert "overlaps" in loom_amd.last_error()
    assert _probs(AT, 5, AT, 6, n=1) == PASSED and _probs(AT, 5, AT + 4, 6, n=1) == loom_amd.ERR_ARG


def test_lora_rows_at_two_strides_lie_apart():
    """At two strides the ranges count: refused where they meet, though rows might pass between each other."""
    assert _lora(AT, 32, None, 64, AT + 4 * 16, 256) == loom_amd.ERR_ARG
    assert _lora(AT, 32, None, 64, AT + 4 * 32 * 4, 256) == PASSED
    assert _lora(AT, 256, None, 64, AT + 4 * (3 * 256 + 32), 64) == PASSED
    assert _lora(AT, 256, None, 64, AT + 4 * (3 * 256 + 31), 64) == loom_amd.ERR_ARG


def _attn(prefix, own, n=1, kv=1, hd=64):
    L = loom_amd.lib()
    return L.loomhip_prefix_attn_dev(C.byref(loom_amd.KvRowsDesc(FAKE, FAKE, *prefix)), C.byref(loom_amd.KvRowsDesc(FAKE, FAKE, *own)),
                                     FAKE, FAKE, None, n, 1, 4, kv, hd, 0.125, FAKE, 0, FAKE, 1 << 40, None)


def test_prefix_attn_strides_of_dimensions_of_one():
    """rows, lane stride, row stride, head stride: what one lane, row or key head has no use for may be anything."""
    fine = (16, 0, 128, 64)
    assert _attn((16, 3, 128, 7), (8, 1029, 128, 12)) == PASSED                # a key head
    assert _attn((1, 3, 7, 64), (1, 1024, 1 << 30, 64), n=2, kv=2) == PASSED   # a row
    assert _attn(fine, (8, 1029, 128, 64), kv=2) == PASSED                     # a lane
    for prefix, own, n, kv in (((16, 0, 127, 64), fine, 1, 1), (fine, (8, 1024, 132, 64), 1, 1), (fine, (8, 1029, 128, 64), 2, 1),
                               ((16, 0, 128, 60), fine, 1, 2), (fine, (8, 1024, 128, 60), 1, 2),
                               ((2, 0, 1 << 24, 64), fine, 1, 1)):
        assert _attn(prefix, own, n, kv) == loom_amd.DECLINED
    assert _attn((2, 0, 32, 64), fine) == loom_amd.ERR_ARG


def test_prefix_attn_keys_without_values():
    from loom_amd import serving

    q, kp, ko = torch.zeros(2, 1, 4, 64), torch.zeros(8, 2, 64).half(), torch.zeros(2, 8, 2, 64).half()
    ln = torch.ones(2, dtype=torch.int32)
    for args in ((kp, None, ko, ko), (None, kp, ko, ko), (kp, kp, ko, None), (kp, kp, None, ko), (None, kp, None, ko)):
        with pytest.raises(ValueError, match="keys without values"):
            serving.prefix_attn_dev(q, *args, ln, 1.0)


def test_prefix_attn_limits():
    """n * n_q * n_heads up to 2^25, cache rows below 2^30, work items below 2^24."""
    L = loom_amd.lib()

    def call(n, nq, heads, kv, own=8, prefix=16):
        kvs = (loom_amd.KvRowsDesc(FAKE, FAKE, rows, 0, kv * 64, 64) for rows in (prefix, own))
        return L.loomhip_prefix_attn_dev(*map(C.byref, kvs), FAKE, FAKE, None, n, nq, heads, kv, 64, 0.125, FAKE, 0, FAKE,
                                         1 << 50, None)

    assert call(4096, 2048, 4, 2) == PASSED and call(4096, 2049, 4, 2) == loom_amd.DECLINED
    assert call(8192, 4096, 1, 1) == PASSED and call(8192, 4097, 1, 1) == loom_amd.DECLINED
    assert call(2, 1, 4, 2, own=(1 << 30) - 1) == PASSED and call(2, 1, 4, 2, own=1 << 30) == loom_amd.DECLINED
    assert call(2, 1, 4, 2, prefix=(1 << 30) - 1) == PASSED and call(2, 1, 4, 2, prefix=1 << 30) == loom_amd.DECLINED
    assert call(65535, 1, 255, 255, prefix=0) == PASSED and call(65535, 1, 257, 257, prefix=0) == loom_amd.DECLINED


def test_pointers_aligned_to_their_elements():
    """Lengths, ids and scales as well: a uniform load drops an address's low bits."""
    L = loom_amd.lib()
    kv = loom_amd.KvRowsDesc(FAKE, FAKE, 16, 1024, 128, 64)

    def attn(own_len, q_len):
        return L.loomhip_prefix_attn_dev(C.byref(kv), C.byref(kv), FAKE, own_len, q_len, 2, 1, 4, 2, 64, 0.125, FAKE, 0, FAKE,
                                         1 << 40, None)

    def lora(scale, ids):
        d = loom_amd.LoraDesc(loom_amd.F16, 2, 8, 64, 32, FAKE, FAKE, scale)
        return L.loomhip_lora_dev(C.byref(d), AT, 32, ids, None, 64, 4, 2 * AT, 64, FAKE, 1 << 40, None)

    assert attn(FAKE + 4, FAKE + 8) == PASSED and lora(FAKE + 4, FAKE + 8) == PASSED
    for off in (1, 2, 3):
        for rc in (attn(FAKE + off, None), attn(FAKE, FAKE + off), lora(FAKE + off, FAKE), lora(FAKE, FAKE + off)):
            assert rc == loom_amd.ERR_ARG and "aligned" in loom_amd.last_error()
