"""The batched serving operators on the device at values and layouts beside the
ordinary: no number among the logits or in the caches, an infinite temperature,
columns of one buffer, dimensions of one."""
import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving import _attn, _attn_case, _attn_ref, _dev, _lora_case, _lora_ref, _rng, _within, sv  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [700, 5000, 20000, 40001, 151936])
def test_token_probs_rows_with_nan(sv, vocab):
    """At a temperature of zero the pick is the frame's: the first maximum among the numbers, a NaN is passed over.  At
    any other a NaN makes the row NaN, wherever it stands and whatever stands beside it."""
    x = (_rng(8, vocab).standard_normal((9, vocab)) * 2).astype(np.float32)
    t = np.array([0, 0, 0, 0, -1, 1, 0.5, 1, 1], np.float32)
    x[0, 0] = np.nan
    x[1] = np.nan
    x[1, vocab // 3] = -5.0
    x[2] = -np.inf
    x[2, vocab // 2] = np.nan  # nothing above -inf
    x[3, [vocab // 4, vocab // 2]] = 60.0
    x[3, [vocab // 4 - 1, vocab // 4 + 1, vocab - 1]] = np.nan
    x[4, ::2] = np.nan
    x[5, vocab - 1] = np.nan
    x[6, :vocab - vocab // 5] = -np.inf
    x[6, 17] = np.nan  # among -inf alone in its part of a long row
    x[7] = -np.inf
    x[7, vocab // 2] = np.nan
    x[8, :vocab // 2] = -np.inf  # no NaN: a part of -inf alone has no share
    got = sv.token_probs_dev(_dev(x), _dev(t)).cpu().numpy()
    want = np.zeros((5, vocab), np.float32)
    for r in (0, 1, 3, 4):
        want[r, int(np.nanargmax(x[r]))] = 1.0
    assert np.array_equal(got[:5], want)
    assert np.isnan(got[5:8]).all()
    w, bound = ref.token_probs(x[8:], t[8:])
    _within(got[8:], w, bound)


@pytest.mark.parametrize("vocab", [700, 4096, 4097, 20000, 40001, 40960])
def test_token_probs_infinite_temperature(sv, vocab):
    """Every finite logit alike, a masked one still nothing; whatever the vocabulary leaves of its last part."""
    x = (_rng(4, vocab).standard_normal((3, vocab)) * 50).astype(np.float32)
    x[1, vocab // 3:] = -np.inf
    x[2, 1::2] = np.finfo(np.float32).min
    got = sv.token_probs_dev(_dev(x), _dev(np.full(3, np.inf, np.float32))).cpu().numpy().astype(np.float64)
    live = np.isfinite(x)
    want = live / live.sum(1, keepdims=True)
    # exponentials of exactly 1 and their sum, a whole number below 2^24; the division and the last product round.  The
    # exponent of a logit 2^128 below the others is held to 2^-20 of its share.
    bound = want * (2 * ref.EPS + np.array([0.0, 0.0, 2.0 ** -19])[:, None])
    _within(got, want, bound)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lanes", [1, 40])
def test_prefix_attn_cached_value_that_is_no_number(sv, lanes, hd, bad):
    """One element of one value row, its key an ordinary one or of no weight: that column of the rows that see it is NaN,
    wherever the row stands, and nothing else changes."""
    c = _attn_case(8, 2, hd, 300, lanes, 3, 75)
    c["own_len"][:] = 67
    c["q_len"][:] = 3
    want, bound = _attn_ref(c)
    for where, row, first in (("vp", 0, 0), ("vp", 299, 0), ("vp", 130, 0), ("vo", 3, 0), ("vo", 65, 1), ("vo", 66, 2)):
        for weightless in (False, True):
            d = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.items()}
            at = (row, 1, 5) if where == "vp" else (0, row, 1, 5)
            d[where][at] = bad
            w, b = want, bound
            if weightless:  # far below every other score
                d["k" + where[1]][at[:-1]] = 0
                d["k" + where[1]][at[:-2] + (1, slice(0, 8))] = -6e4
                d["q"][..., :8] = np.abs(d["q"][..., :8]) + 1
                w, b = _attn_ref(d | {where: c[where]})
            got = _attn(sv, d).cpu().numpy()
            hit = np.zeros(got.shape, bool)
            hit[slice(None) if where == "vp" else 0, first:, 4:, 5] = True
            assert np.isnan(got[hit]).all(), (where, row, weightless)
            _within(got[~hit], w[~hit], b[~hit], f"{where} {row}")


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefix_attn_cached_key_that_is_no_number(sv, hd, bad):
    """One element of one key row: NaN makes the rows that see it NaN; an infinity does so too, or its score is minus
    infinity and they are what they are without it.  Other key heads and rows that do not see it keep their results."""
    c = _attn_case(8, 2, hd, 150, 3, 2, 40)
    c["own_len"][:] = 33
    c["q_len"][:] = 2
    want, bound = _attn_ref(c)
    c["kp"][77, 1, 3] = bad
    gone = dict(c, kp=np.delete(c["kp"], 77, 0), vp=np.delete(c["vp"], 77, 0))
    without, wbound = _attn_ref(gone)
    got = _attn(sv, c).cpu().numpy()
    _within(got[:, :, :4], want[:, :, :4], bound[:, :, :4], "the other key head")
    for i in range(3):
        for j in range(2):
            for h in range(4, 8):
                if np.isnan(bad) or (c["q"][i, j, h, 3] > 0) == (bad > 0):
                    assert np.isnan(got[i, j, h]).all()
                elif not np.isnan(got[i, j, h]).all():
                    _within(got[i, j, h], without[i, j, h], wbound[i, j, h], "without the key")


def test_lora_columns_of_one_buffer(sv):
    """x, base and out side by side in the rows of one buffer share no element; what lies between them stays."""
    import torch

    for n, rank in ((37, 24), (901, 250)):  # vectors one by one, and tiles of them
        t = _lora_case(n, 200, 128, rank, 5, "f16")
        want, bound = _lora_ref(t)
        wide = torch.full((n, 600), 3.25, device="cuda")
        x, base, out = wide[:, :128], wide[:, 150:350], wide[:, 390:590]
        x.copy_(t["x"])
        base.copy_(t["base"])
        assert sv.lora_dev(x, t["a"], t["b"], t["scale"], t["ids"], base=base, out=out) is out
        _within(out.cpu().numpy(), want, bound)
        assert bool((x == t["x"]).all()) and bool((base == t["base"]).all())
        for gap in (wide[:, 128:150], wide[:, 350:390], wide[:, 590:]):
            assert bool((gap == 3.25).all())


def test_prefix_attn_dimensions_of_one(sv):
    """A cache of one row, one key head or one lane: the stride of that dimension has no part in the layout."""
    import torch

    c = _attn_case(4, 1, 64, 1, 1, 1, 1)
    c["own_len"][:] = 1
    want, bound = _attn_ref(c, q_len=False)

    def odd(name, keep):  # the same values, the strides of the dimensions of one set to `keep`
        a = _dev(c[name])
        return torch.as_strided(a, a.shape, tuple(k if s == 1 else st for s, st, k in zip(a.shape, a.stride(), keep)))

    q, ln = _dev(c["q"]), _dev(c["own_len"])
    for k, v in (((3, 7, 1), (3, 7, 1)), ((5, 64, 1), (64, 64, 1)), ((1 << 24, 12, 1), (0, 0, 1))):
        got = sv.prefix_attn_dev(q, odd("kp", k), odd("vp", v), odd("ko", (9, *k)), odd("vo", (64, *v)), ln, c["scale"])
        _within(got.cpu().numpy(), want, bound, f"{k} {v}")
