"""That the inputs of serving_forms.py reach the kernels they name, and would
show operands of fewer bits, without a GPU."""
import os
import re

import numpy as np
import pytest

import loom_amd
import serving_forms as sf

SOURCE = open(os.path.join(loom_amd.HERE, "csrc", "prefix_attn.hip")).read()


def _rule(name):
    """`p.<name> = c1 ? v1 : c2 ? v2 : v3;` of the plan as a function of its variables."""
    text = re.search(rf"^ *p\.{name} = (.*?);$", SOURCE, re.M).group(1)
    *steps, last = text.split(" : ")
    steps = [s.split(" ? ") for s in steps]
    return lambda **v: next((int(x) for cond, x in steps if eval(cond, {}, v)), int(last))


def _form(shape):
    heads, kv, hd, _, n, nq, _ = shape
    mine = nq * (heads // kv)
    v = {"hd": hd, "mine": mine, "all": n * mine}
    return tuple(_rule(name)(**v) for name in ("hdp", "rwp", "rwo"))


def test_every_form_of_the_attention_kernel_is_reached():
    built = {(hdp, int(a), int(b)) for a, b in re.findall(r"prefix_attn_kernel<HDP, (\d), (\d)>", SOURCE) for hdp in (64, 128, 256)}
    assert built and set(sf.ATTN_FORMS) == built
    for form, (shape, _) in sf.ATTN_FORMS.items():
        assert _form(shape) == form, shape
    assert {_form(s) for s in sf.ATTN_MORE} == {(64, 4, 2), (128, 4, 2), (256, 4, 2)}
    assert _form(sf.ATTN_LONG) == (128, 4, 2)


@pytest.mark.parametrize("form", sf.ATTN_FORMS, ids=str)
def test_prefix_ranges_have_several_tiles(form):
    """From the workspace, which holds a record a row and range: the prefix has no more ranges than that, so its ranges
    are at least this long."""
    (heads, kv, hd, P, n, nq, own), tiles = sf.ATTN_FORMS[form]
    nb = loom_amd.lib().loomhip_prefix_attn_ws(P, own, n, nq, heads, kv, hd)
    slots = (nb - 16) // (n * nq * heads * (hd * 4 + 8))
    ranges = slots - 1  # a lane's own rows are one at least
    hdp, rwp, _ = form
    tile = 32 if (hdp, rwp) == (256, 4) else 4 // rwp * (64 if rwp == 4 else 32)
    length = ((P + ranges - 1) // ranges + 127) // 128 * 128
    assert length // tile >= tiles, (slots, length, tile)


def _shows(want, bound, got):
    ok = ~np.isnan(want)
    return bool((np.abs(got[ok] - want[ok]) > bound[ok]).any())


ATTN_SHAPES = [s for s, _ in sf.ATTN_FORMS.values()] + sf.ATTN_MORE + [sf.ATTN_LONG]


@pytest.mark.parametrize("shape", ATTN_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_with_operands_of_11_bits_is_seen(shape):
    c = sf.attn_case(shape)
    for ragged in (True, False):
        want, bound = sf.attn(c, ragged)
        assert _shows(want, bound, sf.attn(c, ragged, query=sf.f16)[0]), "query"
        assert _shows(want, bound, sf.attn(c, ragged, weights=sf.f16)[0]), "weights"

        def parts(x):  # two of 11 bits
            h = sf.f16(x)
            return h + sf.f16((x - h) * 4096) / 4096

        assert not _shows(want, bound, sf.attn(c, ragged, query=parts, weights=parts)[0])


@pytest.mark.parametrize("shape", sf.LORA_FORMS, ids=lambda s: "x".join(map(str, s)))
def test_adapters_with_operands_of_few_bits_are_seen(shape):
    c = sf.lora_case(shape)
    want, bound = sf.lora(c)
    for few in (sf.f16, sf.bf16):
        assert _shows(want, bound, sf.lora(c, vectors=few)[0]) and _shows(want, bound, sf.lora(c, inner=few)[0])
    assert not _shows(want, bound, sf.lora(c, vectors=lambda x: x.astype(np.float32).astype(np.float64),
                                           inner=lambda y: y.astype(np.float32).astype(np.float64))[0])


def test_every_form_of_the_adapter_kernels_is_reached():
    """In fp16, by the library's own limits: one launch (lanes a row of B_e), two for few vectors (the same, and twice
    eight ranks a lane), tiles (of 16 ranks)."""
    source = open(os.path.join(loom_amd.HERE, "csrc", "lora.hip")).read()
    few_bytes = float(re.search(r"LORA_FEW = ([\de.]+);", source).group(1))
    small = float(re.search(r"LORA_SMALL = ([\de.]+);", source).group(1))
    reached = set()
    for n, rows, cols, rank, _ in sf.LORA_FORMS:
        d = loom_amd.LoraDesc(loom_amd.F16, 1, rank, rows, cols)
        step = next(i for i, most in enumerate((8, 16, 32, 64, 128, 256)) if rank <= most)
        few = n <= 65535 and n * rank * (rows + cols) * 2 <= few_bytes
        one = few and rank <= 64 and rank * cols * 2 <= small
        assert one == (loom_amd.lib().loomhip_lora_ws(d, n) == 0)
        reached.add(("one", step) if one else ("few", step) if few else ("many", max(step, 1)))
    assert reached == {("one", s) for s in range(4)} | {("few", s) for s in range(6)} | {("many", s) for s in range(1, 6)}
