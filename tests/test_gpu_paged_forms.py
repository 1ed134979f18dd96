"""Every form of the attention over pages on the device: each row seen once, the
row that outweighs all others found wherever it stands, queries and weights held
in all of their parts (paged_forms.py; test_paged_forms.py shows what these
inputs catch)."""
import numpy as np
import pytest

import paged_forms as pf

pytestmark = pytest.mark.gpu
KINDS = ["f16", "bf16"]


def _id(form):
    return "-".join(map(str, form))


@pytest.fixture(scope="module")
def sv():
    import loom_amd
    from loom_amd import serving

    loom_amd.init(0)
    return serving


class _On:
    """A case on the device."""

    def __init__(self, sv, form, c, kind):
        import torch

        self.sv, self.c = sv, c
        dt = torch.float16 if kind == "f16" else torch.bfloat16
        self.k, self.v = (torch.from_numpy(x).cuda().to(dt) for x in (c.k, c.v))
        assert (self.k.float().cpu().numpy() == c.k).all() and (self.v.float().cpu().numpy() == c.v).all()
        # a table as wide as the longest lane where its width decides on the form
        self.table = torch.from_numpy(np.ascontiguousarray(c.table[:, :-1] if form[0] == "whole" else c.table)).cuda()
        self.lens = torch.tensor(c.lens, dtype=torch.int32, device="cuda")

    def run(self, window=0):
        import torch

        out = self.sv.paged_attn_dev(torch.from_numpy(self.c.q).cuda(), self.k, self.v, self.table, self.lens, 1.0, window=window)
        return out.double().cpu().numpy()


def _within(got, want, bound, what):
    off = np.abs(got - want) - bound
    assert np.isfinite(got).all() and off.max() <= 0, (what, np.unravel_index(off.argmax(), off.shape), off.max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_every_row_is_seen_once(sv, form, kind):
    shape = pf.FORMS[form]
    for by in (1, shape[2]):
        c = pf.coverage_case(shape, by)
        on = _On(sv, form, c, kind)
        for window in (0, 1, 200, 1000, 5001):
            _within(on.run(window), *pf.coverage(c, by, window), (by, window))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_the_row_that_outweighs_all_others(sv, form, kind):
    c = pf.edge_case(pf.FORMS[form])
    on = _On(sv, form, c, kind)
    for window in (0, 200, 3000):
        for turn in range(12 if len(c.lens) < 10 else 3):
            want = pf.edges(c, pf.edge_rows(c, turn, window))
            assert (on.run(window) == want).all(), (window, turn)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_queries_and_weights_are_held_in_all_their_parts(sv, form, kind):
    c = pf.query_case(pf.FORMS[form])
    _within(_On(sv, form, c, kind).run(), *pf.query(c, kind), "queries")
    c = pf.weight_case(pf.FORMS[form])
    on = _On(sv, form, c, kind)
    live = np.array(c.lens) > 0
    for turn in range(pf.WEIGHT_TURNS):
        pf.weight_queries(c, turn)
        got = on.run()
        assert (got[~live] == 0).all()
        _within(got[live], 1.0, pf.WEIGHTS_BOUND, ("weights", turn))
