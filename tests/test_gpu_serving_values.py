"""The batched serving operators on the device at values and layouts beside the
ordinary: no number among the logits of a greedy row."""
import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving import _dev, _rng, _within, sv  # noqa: F401

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
