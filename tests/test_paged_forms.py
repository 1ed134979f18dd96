"""That the inputs of paged_forms.py reach the kernels they name, and would show
a row that is missing, doubled or another's and operands of fewer parts, without
a GPU."""
import numpy as np
import pytest

import loom_amd
import paged_forms as pf


def _id(form):
    return "-".join(map(str, form))


@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_every_form_is_reached(form):
    """From the workspace: none for whole lanes, otherwise the records that decide how many waves join them; and that some
    lane is cut, as the plan cuts."""
    H, KV, hd, ps, lens = pf.FORMS[form]
    launch, head_class, once = form
    rows = (max(-(-x // ps) for x in lens) + 1) * ps
    group, n = H // KV, len(lens)
    blocks = -(-group // 16)
    assert (blocks == 1) == once and head_class == (64 if hd <= 64 else 128 if hd <= 128 else 256)
    # the whole form's tables: lens in a table as wide as the tests', with its entry of no page
    nb = loom_amd.lib().loomhip_paged_attn_ws(rows if launch != "whole" else max(lens), n, H, KV, hd)
    if launch == "whole":
        assert nb == 0
        return
    room = 256 if hd > 128 else 512
    records = (nb - 16) // (8 + min(group, 16) * (hd * 4 + 8))
    assert records == {2: room, 1: 4 * room}[launch]
    items, unit = KV * blocks, 256 if hd <= 64 else 128
    u = -(-np.array(lens) // unit)
    share = -(-int(u.sum()) * items // room)
    pieces = lambda L: np.maximum(1, -(-u // L))
    cuts = [max(1, -(-share * s // 16)) for s in (16, 17, 18, 20, 24, 32)]
    L = next((x for x in cuts if pieces(x).sum() * items <= room), max(1, (share + 1) // 2))
    assert pieces(L).max() > 1


def _shown(want, bound, got):
    return bool((np.abs(got - want) > bound).any())


@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_a_row_missing_doubled_or_anothers_is_shown(form):
    shape = pf.FORMS[form]
    r = np.random.default_rng(3)
    by_one, by_head = (pf.coverage_case(shape, by) for by in (1, shape[2]))
    for window in (0, 200):
        i = int(np.argmax(shape[4]))
        T, first = shape[4][i], by_one.first(i, window)
        for t in (first, T - 1, *r.integers(first, T, 3)):
            other = int(r.integers(first, T))
            for planted in (dict(without=[(i, t)]), dict(twice=[(i, t)]),
                            dict(without=[(i, t)], twice=[(i, t + 1 if t < T - 1 else t - 1)]),
                            dict(without=[(i, t)], twice=[(i, other)]) if other != t else dict(without=[(i, t)])):
                shown = [_shown(*pf.coverage(c, by, window), pf.coverage(c, by, window, **planted)[0])
                         for c, by in ((by_one, 1), (by_head, shape[2]))]
                # two rows that both choices put in one column each stand for one another
                same = planted.get("twice") and planted.get("without") and all(
                    pf.coverage_column(c, i, 0, t, by) == pf.coverage_column(c, i, 0, planted["twice"][0][1], by)
                    for c, by in ((by_one, 1), (by_head, shape[2])))
                assert any(shown) or same, (window, planted)


@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_edge_rows_are_the_only_ones_with_weight(form):
    c = pf.edge_case(pf.FORMS[form])
    for window in (0, 200):
        at = pf.edge_rows(c, 0, window)
        pf.edges(c, at)  # asserts the distance to every other row
        assert ((at >= 0) == (np.array(c.lens) > 0)[:, None]).all()
        for i, T in enumerate(c.lens):
            assert not T or (at[i, 0] == c.first(i, window) and (c.H < 2 or at[i, 1] == T - 1))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("form", pf.FORMS, ids=_id)
def test_operands_of_fewer_parts_are_shown(form, kind):
    bits, parts = pf.BITS[kind]
    c = pf.query_case(pf.FORMS[form])
    want, bound = pf.query(c, kind)
    assert not _shown(want, bound, pf.query(c, kind, pf.in_parts(bits, parts))[0])
    assert _shown(want, bound, pf.query(c, kind, pf.in_parts(bits, parts - 1))[0])
    c = pf.weight_case(pf.FORMS[form])
    live = np.repeat(np.array(c.lens)[:, None] > 0, c.H, 1)
    off = {parts: 0.0, parts - 1: 0.0}
    for turn in range(pf.WEIGHT_TURNS):
        pf.weight_queries(c, turn)
        for p in off:
            off[p] = max(off[p], np.abs(pf.weights(c, pf.in_parts(bits, p))[live] - 1).max())
    assert off[parts] <= 2 * pf.EPS and off[parts - 1] > 1.5 * pf.WEIGHTS_BOUND
