"""The batched serving operators on the device against their definitions in 64
bits (serving_ref.py, elementwise error bounds derived there), at the sizes,
masks, strides and values where they can go wrong, and together."""

import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sv():
    import loom_amd
    from loom_amd import serving

    loom_amd.init(0)
    return serving


def _rng(*key):
    return np.random.default_rng([int(k) for k in key])


def _dev(a, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    ok = ~np.isnan(want)
    off = np.abs(got[ok] - want[ok]) - bound[ok]
    assert np.isfinite(got[ok]).all(), what
    assert off.size == 0 or off.max() <= 0, f"{what}: {off.max()} over the bound, {np.abs(got[ok] - want[ok]).max()} off"


# ---- shared-prefix attention ------------------------------------------------------


def _attn_case(heads, kv, hd, prefix, n, nq, own, seed=1, q_scale=1.0):
    r = _rng(heads, kv, hd, prefix, n, nq, own, seed)
    c = {"q": (r.standard_normal((n, nq, heads, hd)) * q_scale).astype(np.float32),
         "kp": r.standard_normal((prefix, kv, hd)).astype(np.float16),
         "vp": r.standard_normal((prefix, kv, hd)).astype(np.float16),
         "ko": r.standard_normal((n, own, kv, hd)).astype(np.float16),
         "vo": r.standard_normal((n, own, kv, hd)).astype(np.float16),
         "own_len": r.integers(0, own + 1, n).astype(np.int32),
         "q_len": r.integers(0, nq + 1, n).astype(np.int32), "scale": 1.0 / np.sqrt(hd)}
    c["own_len"][-1] = own
    c["q_len"][-1] = nq
    return c


def _attn(sv, c, q_len=True, out=None):
    args = [_dev(c[k]) for k in ("q", "kp", "vp", "ko", "vo", "own_len")]
    return sv.prefix_attn_dev(*args, c["scale"], q_len=_dev(c["q_len"]) if q_len else None, out=out)


def _attn_ref(c, q_len=True):
    return ref.prefix_attn(c["q"], c["kp"], c["vp"], c["ko"], c["vo"], c["own_len"], c["q_len"] if q_len else None, c["scale"])


ATTN = [
    # heads, kv, hd, prefix, n, nq, own
    (1, 1, 8, 1, 1, 1, 1),
    (4, 2, 64, 0, 2, 1, 5),       # no prefix
    (6, 6, 48, 33, 3, 2, 17),     # every head its own keys
    (8, 1, 128, 129, 1, 1, 1),    # one key head, one own row
    (32, 4, 128, 700, 3, 5, 40),
    (32, 4, 128, 64, 33, 1, 64),
    (8, 2, 256, 65, 2, 3, 9),
    (24, 8, 96, 255, 4, 4, 31),
    (12, 1, 40, 63, 7, 1, 130),
    (71, 1, 64, 300, 2, 2, 3),    # a group wider than a tile
    (3, 3, 72, 31, 1, 9, 9),      # all own rows are drafts
    (16, 2, 200, 127, 2, 2, 66),
    (2, 1, 128, 2500, 1, 1, 1500),
    (40, 8, 128, 1025, 17, 3, 257),
    (4, 4, 32, 5000, 2, 1, 1),
]


@pytest.mark.parametrize("shape", ATTN, ids=lambda s: "x".join(map(str, s)))
def test_prefix_attn_matches_its_definition(sv, shape):
    c = _attn_case(*shape)
    want, bound = _attn_ref(c, q_len=False)
    _within(_attn(sv, c, q_len=False).cpu().numpy(), want, bound, "every query")
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound, "ragged")
    assert (got[np.isnan(want)] == 0).all()


@pytest.mark.parametrize("shape", [(2, 1, 8, 20, 300, 2, 9), (2, 2, 16, 0, 1030, 3, 4), (1, 1, 16, 70, 1, 1500, 1500),
                                   (4, 2, 32, 200, 600, 1, 5)], ids=lambda s: "x".join(map(str, s)))
def test_prefix_attn_many_lanes_and_queries(sv, shape):
    c = _attn_case(*shape)
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound, "ragged")
    assert (got[np.isnan(want)] == 0).all()
    c["q_len"][:-1] = 0  # one lane alone has query tokens
    want, bound = _attn_ref(c)
    _within(_attn(sv, c).cpu().numpy(), want, bound, "one lane")


@pytest.mark.parametrize("scale", [-0.25, 0.0, -3e4])
def test_prefix_attn_scales(sv, scale):
    """A negative scale turns the order around, zero weighs every row alike."""
    c = _attn_case(8, 2, 64, 150, 3, 2, 40)
    c["scale"] = scale
    want, bound = _attn_ref(c)
    _within(_attn(sv, c).cpu().numpy(), want, bound)


def test_prefix_attn_leaves_rows_past_q_len(sv):
    import torch

    c = _attn_case(8, 2, 64, 40, 5, 4, 20)
    out = torch.full((5, 4, 8, 64), 7.5, device="cuda")
    got = _attn(sv, c, out=out)
    assert got is out
    want, bound = _attn_ref(c)
    g = out.cpu().numpy()
    _within(g, want, bound)
    assert (g[np.isnan(want)] == 7.5).all() and np.isnan(want).any()


@pytest.mark.parametrize("prefix", [0, 1, 64, 200])
def test_prefix_attn_rows_that_see_little(sv, prefix):
    """Lengths of zero and one, lengths below the number of queries (the first queries see no own row; without a
    prefix nothing at all: zero), lengths and counts out of range (clamped)."""
    c = _attn_case(8, 2, 64, prefix, 8, 3, 70)
    c["own_len"] = np.array([0, 1, 2, 3, 70, 71, 1 << 30, -5], np.int32)
    c["q_len"] = np.array([3, 3, 3, 3, 100, 1, 0, 3], np.int32)
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound)
    if prefix == 0:
        assert (got[0] == 0).all() and (got[1, :2] == 0).all() and (got[7] == 0).all()


def test_prefix_attn_without_own_rows(sv):
    c = _attn_case(8, 2, 64, 100, 3, 2, 1)
    c["own_len"][:] = 0
    want, bound = _attn_ref(c, q_len=False)
    got = sv.prefix_attn_dev(_dev(c["q"]), _dev(c["kp"]), _dev(c["vp"]), None, None, None, c["scale"])
    _within(got.cpu().numpy(), want, bound)
    c = _attn_case(8, 2, 64, 0, 3, 2, 30)
    want, bound = _attn_ref(c, q_len=False)
    got = sv.prefix_attn_dev(_dev(c["q"]), None, None, _dev(c["ko"]), _dev(c["vo"]), _dev(c["own_len"]), c["scale"])
    _within(got.cpu().numpy(), want, bound)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefix_attn_rows_behind_hold_anything(sv, bad, hd):
    """Rows past a lane's length, and a later draft's rows for the query before it, have no part in the result."""
    c = _attn_case(8, 2, hd, 90, 4, 3, 75)
    c["own_len"] = np.array([0, 10, 40, 67], np.int32)
    c["q_len"] = np.array([3, 3, 2, 3], np.int32)
    want, bound = _attn_ref(c)
    for i, ln in enumerate(c["own_len"]):
        c["ko"][i, ln:] = bad
        c["vo"][i, ln:] = bad
    _within(_attn(sv, c).cpu().numpy(), want, bound, "behind the length")
    # the last drafted row: only the last query sees it, the others' results stay
    for i, ln in enumerate(c["own_len"]):
        if ln:
            c["ko"][i, ln - 1] = bad
            c["vo"][i, ln - 1] = bad
    got = _attn(sv, c).cpu().numpy()
    for i, (ln, L) in enumerate(zip(c["own_len"], c["q_len"])):
        if ln:
            _within(got[i, :L - 1], want[i, :L - 1], bound[i, :L - 1], f"lane {i}")
            assert np.isnan(got[i, L - 1]).all()


@pytest.mark.parametrize("hd", [8, 48, 200, 256])
def test_prefix_attn_zeroes_the_rest_of_its_own_output(sv, hd):
    """Rows past q_len of an out made here, over memory that held something else."""
    import torch

    c = _attn_case(4, 2, hd, 33, 9, 3, 12)
    c["q_len"] = np.array([0, 1, 2, 3, 0, 1, 2, 3, 1], np.int32)
    want, bound = _attn_ref(c)
    for _ in range(3):
        torch.full((9, 3, 4, hd), float("nan"), device="cuda")  # freed: the next output's memory
        got = _attn(sv, c).cpu().numpy()
        _within(got, want, bound)
        assert (got[np.isnan(want)] == 0).all() and np.isnan(want).any()


def test_prefix_attn_one_bad_lane_stays_alone(sv):
    c = _attn_case(8, 2, 64, 90, 6, 2, 33)
    c["own_len"][:] = 33
    want, bound = _attn_ref(c, q_len=False)
    c["q"][2, 1, 3] = np.nan
    c["vo"][4, 5] = np.inf
    got = _attn(sv, c, q_len=False).cpu().numpy()
    for i in (0, 1, 3, 5):
        _within(got[i], want[i], bound[i], f"lane {i}")
    _within(got[2, 0], want[2, 0], bound[2, 0])
    _within(np.delete(got[2, 1], 3, 0), np.delete(want[2, 1], 3, 0), np.delete(bound[2, 1], 3, 0))
    assert np.isnan(got[2, 1, 3]).all()
    assert not np.isfinite(got[4]).any()


@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e6, 1e30])
def test_prefix_attn_query_sizes(sv, q_scale):
    """Queries far outside fp16's range: with the scale that brings the scores back."""
    c = _attn_case(8, 2, 64, 90, 2, 2, 33, q_scale=q_scale)
    c["scale"] = float(np.float32(c["scale"] / q_scale)) if q_scale else c["scale"]
    want, bound = _attn_ref(c, q_len=False)
    _within(_attn(sv, c, q_len=False).cpu().numpy(), want, bound)


def test_prefix_attn_mixed_query_sizes(sv):
    """One lane's query a thousand times another's, and scores far apart: a weight of one, the rest of nothing."""
    c = _attn_case(8, 2, 64, 200, 4, 1, 33)
    c["q"] *= np.array([1e-3, 1.0, 30.0, 1e3], np.float32)[:, None, None, None]
    want, bound = _attn_ref(c, q_len=False)
    _within(_attn(sv, c, q_len=False).cpu().numpy(), want, bound)


def test_prefix_attn_strides(sv):
    """A Decoder's caches at one layer (int16 bits, lanes far apart), a prefix inside one of its lanes, and caches with
    the key heads first."""
    import torch

    c = _attn_case(8, 2, 64, 100, 3, 2, 40)
    want, bound = _attn_ref(c)
    k = torch.full((4, 3, 120, 2 * 64), -1, dtype=torch.int16, device="cuda")  # -1: NaN bits
    v = k.clone()
    k[1:, 1, :40], v[1:, 1, :40] = (_dev(c[x]).view(torch.int16).flatten(2) for x in ("ko", "vo"))
    k[0, 1, :100], v[0, 1, :100] = (_dev(c[x]).view(torch.int16).flatten(1) for x in ("kp", "vp"))
    args = [t[0, 1, :100].unflatten(-1, (2, 64)) for t in (k, v)] + [t[1:, 1, :40].unflatten(-1, (2, 64)) for t in (k, v)]
    got = sv.prefix_attn_dev(_dev(c["q"]), *args, _dev(c["own_len"]), c["scale"], q_len=_dev(c["q_len"]))
    _within(got.cpu().numpy(), want, bound, "frame caches")
    args = [_dev(c[x].transpose(1, 0, 2)).transpose(0, 1) for x in ("kp", "vp")]
    args += [_dev(c[x].transpose(0, 2, 1, 3)).transpose(1, 2) for x in ("ko", "vo")]
    got = sv.prefix_attn_dev(_dev(c["q"]), *args, _dev(c["own_len"]), c["scale"], q_len=_dev(c["q_len"]))
    _within(got.cpu().numpy(), want, bound, "heads first")


def test_prefix_attn_refuses_unaligned_rows(sv):
    import torch

    import loom_amd

    q, ln = torch.zeros(2, 1, 4, 64, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 8, 2, 68, dtype=torch.float16, device="cuda")
    loom_amd.take_launch_count()
    for kk in (k[..., :64], k.view(-1)[4:4 + 2 * 7 * 2 * 64].view(2, 7, 2, 64)):
        with pytest.raises(loom_amd.LoomHipError):
            sv.prefix_attn_dev(q, None, None, kk, kk, ln, 1.0)
    assert loom_amd.take_launch_count() == 0


def test_prefix_attn_beyond_32_bit_offsets(sv):
    """Lanes 2^30 elements apart and a prefix whose rows are 2^22 apart: offsets past 2^31."""
    import torch

    c = _attn_case(4, 1, 64, 600, 4, 1, 70)
    want, bound = _attn_ref(c, q_len=False)
    big = torch.empty((1 << 32) + (1 << 20), dtype=torch.float16, device="cuda")
    own = big.as_strided((4, 70, 1, 64), (1 << 30, 64, 64, 1))
    pre = big.as_strided((600, 1, 64), (1 << 22, 64, 1), 1 << 16)
    own.copy_(_dev(c["ko"]))
    pre.copy_(_dev(c["kp"]))
    c["vo"], c["vp"] = c["ko"], c["kp"]
    want, bound = _attn_ref(c, q_len=False)
    got = sv.prefix_attn_dev(_dev(c["q"]), pre, pre, own, own, _dev(c["own_len"]), c["scale"])
    _within(got.cpu().numpy(), want, bound)


def test_prefix_attn_agrees_with_the_seam_attention(sv):
    """The engine's attention of one sequence (attnHeads, the host's order) over the same rows in one cache."""
    from loom_amd import backend as be

    heads, kv, hd, prefix, own = 8, 2, 64, 50, 14
    c = _attn_case(heads, kv, hd, prefix, 1, 1, own)
    assert be.attnInit(1, 128, kv * hd)
    for p in range(prefix + own):
        k, v = (c["kp"][p], c["vp"][p]) if p < prefix else (c["ko"][0, p - prefix], c["vo"][0, p - prefix])
        assert be.kvAppend(0, p, k.astype(np.float32).ravel(), v.astype(np.float32).ravel())
    seam = np.empty(heads * hd, np.float32)
    assert be.attnHeads(0, prefix + own - 1, c["q"].ravel(), seam, heads, kv, hd, float(np.float32(c["scale"])))
    be.releaseKvCache()
    got = _attn(sv, c, q_len=False).cpu().numpy()
    want, bound = _attn_ref(c, q_len=False)
    _within(seam.reshape(want.shape), want, bound, "seam")
    _within(got, want, bound)


# ---- adapters -------------------------------------------------------------------


def _lora_case(n, rows, cols, rank, adapters, dtype, seed=1):
    import torch

    r = _rng(n, rows, cols, rank, adapters, seed)
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    t = {"x": _dev(r.standard_normal((n, cols)).astype(np.float32)), "base": _dev(r.standard_normal((n, rows)).astype(np.float32)),
         "a": _dev((r.standard_normal((adapters, rank, cols)) / np.sqrt(cols)).astype(np.float32), dt),
         "b": _dev((r.standard_normal((adapters, rows, rank)) / np.sqrt(rank)).astype(np.float32), dt),
         "scale": _dev(r.uniform(-2, 2, adapters).astype(np.float32)),
         "ids": _dev(r.integers(-1, adapters + 1, n).astype(np.int32))}
    return t


def _lora_ref(t, base=True):
    a = {k: v.float().cpu().numpy() for k, v in t.items()}
    return ref.lora(a["x"], a["a"], a["b"], a["scale"], a["ids"], a["base"] if base else None)


LORA = [
    # n, rows, cols, rank, adapters
    (1, 1, 1, 1, 1),
    (1, 64, 32, 8, 1),
    (1, 4096, 2048, 16, 3),
    (2, 33, 257, 3, 4),
    (15, 100, 96, 16, 2),
    (16, 288, 768, 32, 5),
    (17, 1003, 130, 9, 40),
    (33, 512, 1000, 64, 7),
    (64, 65, 4096, 128, 3),
    (5, 130, 70, 256, 6),
    (130, 16, 2050, 20, 2),
    (300, 260, 288, 12, 9),
    (513, 1024, 512, 48, 33),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", LORA, ids=lambda s: "x".join(map(str, s)))
def test_lora_matches_its_definition(sv, shape, dtype):
    t = _lora_case(*shape, dtype)
    want, bound = _lora_ref(t)
    got = sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=t["base"])
    _within(got.cpu().numpy(), want, bound)
    none = (t["ids"] < 0) | (t["ids"] >= shape[4])
    assert bool((got[none] == t["base"][none]).all())
    want, bound = _lora_ref(t, base=False)
    _within(sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"]).cpu().numpy(), want, bound, "no base")
    out = t["base"].clone()
    assert sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=out, out=out) is out
    assert bool((out == got).all())  # in place: the same kernels, the same bits


LORA_LONG = [
    # two launches, a vector at a time
    (3, 70, 16400, 16, 2),
    (2, 65, 32801, 8, 2),
    (9, 130, 4099, 40, 3),
    (4, 1001, 3000, 64, 3),
    # tiles of vectors that share an adapter
    (700, 131, 321, 256, 5),
    (6001, 333, 517, 16, 7),
    (9001, 500, 700, 8, 3),
    (3001, 400, 500, 33, 40),
    (1203, 301, 402, 100, 4),
    (70000, 3, 5, 1, 3),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("spans", [False, True])
@pytest.mark.parametrize("shape", LORA_LONG, ids=lambda s: "x".join(map(str, s)))
def test_lora_many_vectors_and_long_rows(sv, shape, spans, dtype):
    """Adapters named in any order, and by runs of vectors (the last run none)."""
    import torch

    n, adapters = shape[0], shape[4]
    t = _lora_case(*shape, dtype)
    if spans:
        t["ids"] = (torch.arange(n, device="cuda") * (adapters + 1) // n).to(torch.int32)
    want, bound = _lora_ref(t)
    got = sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=t["base"])
    _within(got.cpu().numpy(), want, bound)
    none = (t["ids"] < 0) | (t["ids"] >= adapters)
    assert bool((got[none] == t["base"][none]).all())
    out = t["base"].clone()
    sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=out, out=out)
    assert bool((out == got).all())
    got = sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"])
    _within(got.cpu().numpy(), *_lora_ref(t, base=False), "no base")


def test_lora_many_vectors_strided(sv):
    """Rows shifted by an odd number of values and by four; what lies beside them stays."""
    import torch

    t = _lora_case(901, 200, 256, 250, 5, "f16")
    want, bound = _lora_ref(t)
    for shift in (1, 4):
        x = torch.full((901, 300), float("nan"), device="cuda")
        x[:, shift:shift + 256] = t["x"]
        wide = torch.full((901, 404), 3.25, device="cuda")
        wide[:, shift:shift + 200] = t["base"]
        view = wide[:, shift:shift + 200]
        sv.lora_dev(x[:, shift:shift + 256], t["a"], t["b"], t["scale"], t["ids"], base=view, out=view)
        _within(view.cpu().numpy(), want, bound, f"shift {shift}")
        assert bool((wide[:, :shift] == 3.25).all()) and bool((wide[:, shift + 200:] == 3.25).all())


def test_lora_many_vectors_bad_values_stay_alone(sv):
    import torch

    t = _lora_case(1500, 220, 240, 128, 4, "bf16")
    t["ids"] = (torch.arange(1500, device="cuda") % 4).to(torch.int32)
    want, bound = _lora_ref(t)
    t["a"][2] = float("nan")
    t["b"][1] = float("inf")
    t["x"][[3, 800]] = float("nan")
    got = sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=t["base"]).cpu().numpy()
    i = np.arange(1500)
    fine = np.isin(i % 4, (0, 3)) & ~np.isin(i, (3, 800))
    _within(got[fine], want[fine], bound[fine])
    assert not np.isfinite(got[i % 4 == 2]).any() and not np.isfinite(got[[3, 800]]).any()


@pytest.mark.parametrize("n", [1, 40, 300])
def test_lora_spans_and_one_adapter(sv, n):
    """Tokens of a request one after the other; every token the same adapter; no token an adapter."""
    import torch

    t = _lora_case(n, 200, 320, 16, 6, "f16")
    for ids in (torch.arange(n, device="cuda") * 6 // max(n, 1), torch.full((n,), 5, device="cuda"),
                torch.full((n,), -1, device="cuda"), torch.full((n,), 1 << 30, device="cuda")):
        t["ids"] = ids.to(torch.int32)
        want, bound = _lora_ref(t)
        got = sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=t["base"])
        _within(got.cpu().numpy(), want, bound)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_lora_strided_rows(sv, dtype):
    """x, base and out as columns of wider matrices (a fused q/k/v output), shifted by an odd number of values; what
    lies beside them stays."""
    import torch

    t = _lora_case(37, 200, 128, 24, 5, dtype)
    want, bound = _lora_ref(t)
    for shift in (1, 4):
        x = torch.full((37, 300), float("nan"), device="cuda")
        x[:, shift:shift + 128] = t["x"]
        wide = torch.full((37, 701), 3.25, device="cuda")
        wide[:, shift:shift + 200] = t["base"]
        view = wide[:, shift:shift + 200]
        sv.lora_dev(x[:, shift:shift + 128], t["a"], t["b"], t["scale"], t["ids"], base=view, out=view)
        _within(view.cpu().numpy(), want, bound, f"shift {shift}")
        assert bool((wide[:, :shift] == 3.25).all()) and bool((wide[:, shift + 200:] == 3.25).all())


def test_lora_adapters_not_used_hold_anything(sv):
    """An adapter of NaN changes the vectors that name it and no other, a vector of NaN itself alone."""
    import torch

    t = _lora_case(50, 70, 96, 16, 4, "bf16")
    t["ids"] = (torch.arange(50, device="cuda") % 4).to(torch.int32)
    want, bound = _lora_ref(t)
    t["a"][2] = float("nan")
    t["b"][1] = float("inf")
    t["x"][3] = float("nan")
    got = sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=t["base"]).cpu().numpy()
    fine = np.array([i % 4 in (0, 3) and i != 3 for i in range(50)])
    _within(got[fine], want[fine], bound[fine])
    assert not np.isfinite(got[[i % 4 == 2 for i in range(50)]]).any()
    assert not np.isfinite(got[3]).any()


def test_lora_large_values(sv):
    """Activations outside fp16's and bf16's comfortable ranges stay f32."""
    t = _lora_case(20, 64, 256, 16, 3, "f16")
    t["x"] *= 1e20
    t["base"] *= 1e20
    t["x"][:, ::2] *= 1e-30
    want, bound = _lora_ref(t)
    _within(sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=t["base"]).cpu().numpy(), want, bound)


# ---- probabilities ----------------------------------------------------------------


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 5), (3, 257), (1, 2048), (2, 2049), (1, 32000), (5, 49999), (70, 1000),
                                        (2, 151936), (1500, 33), (7, 151937), (3, 1024), (2, 1025), (2, 4096), (1, 4097),
                                        (3, 16384), (2, 16385), (1, 32768), (2, 32769), (70, 50257), (200, 40001),
                                        (300, 40003)])
def test_token_probs_matches_its_definition(sv, rows, vocab):
    r = _rng(rows, vocab)
    x = (r.standard_normal((rows, vocab)) * 4).astype(np.float32)
    t = r.uniform(0.3, 2.0, rows).astype(np.float32)
    x[0, vocab // 2] = 30.0
    for temp in (None, t):
        want, bound = ref.token_probs(x, temp)
        got = sv.token_probs_dev(_dev(x), None if temp is None else _dev(temp))
        _within(got.cpu().numpy(), want, bound)
    logits = _dev(x)
    assert sv.token_probs_dev(logits, _dev(t), out=logits) is logits
    assert bool((logits == got).all())  # in place: the same bits


@pytest.mark.parametrize("vocab", [5000, 4900, 1001, 40001])
def test_token_probs_special_rows(sv, vocab):
    """Masked values (-inf and the type's lowest), a row of them alone, temperatures of zero, below, NaN, tiny, huge."""
    r = _rng(5)
    x = (r.standard_normal((12, vocab)) * 2).astype(np.float32)
    x[0, 100:vocab - 100] = -np.inf
    x[1, 100:] = np.finfo(np.float32).min
    x[2] = -np.inf
    x[2, vocab - 679] = -3.0
    x[3] = -np.inf
    x[4] = np.finfo(np.float32).min
    x[5] = 1e30
    x[6, [50, vocab - 500, vocab - 100]] = 99.0  # the maximum three times
    x[7, [50, vocab - 500, vocab - 100]] = 99.0
    x[8, vocab - 1] = 99.0
    x[11] = -np.inf
    t = np.ones(12, np.float32)
    t[6], t[7], t[8], t[9], t[10], t[11] = 0.0, -1.0, np.nan, 1e-3, 1e6, 0.0
    want, bound = ref.token_probs(x, t)
    got = sv.token_probs_dev(_dev(x), _dev(t)).cpu().numpy()
    _within(got, want, bound)
    assert (got[3] == 0).all() and got[2, vocab - 679] == 1 and (got[11] == 0).all()
    for row, at in ((6, 50), (7, 50), (8, vocab - 1)):
        assert got[row, at] == 1 and got[row].sum() == 1
    x[0, 7], x[1, 7], x[3] = np.nan, np.inf, np.nan
    got = sv.token_probs_dev(_dev(x), _dev(t)).cpu().numpy()
    assert np.isnan(got[[0, 1, 3]]).all()
    fine = [2, 4, 5, 6, 7, 8, 9, 10, 11]
    _within(got[fine], want[fine], bound[fine])


@pytest.mark.parametrize("vocab", [700, 33000])
def test_token_probs_strided_rows(sv, vocab):
    import torch

    import loom_amd
    from loom_amd.backend import _ptr, _stream

    x = (_rng(9).standard_normal((6, vocab)) * 3).astype(np.float32)
    wide = torch.full((6, vocab + 201), float("nan"), device="cuda")
    wide[:, 3:vocab + 3] = _dev(x)
    out = torch.full((6, vocab + 111), 5.0, device="cuda")
    L = loom_amd.lib()
    nb = L.loomhip_token_probs_ws(6, vocab)
    ws = torch.empty(max(nb, 16), dtype=torch.uint8, device="cuda")
    src, dst = wide[:, 3:], out[:, 1:]
    assert L.loomhip_token_probs_dev(_ptr(src), 6, vocab, vocab + 201, None, _ptr(dst), vocab + 111, _ptr(ws), nb,
                                     _stream()) == 0
    want, bound = ref.token_probs(x, None)
    _within(out[:, 1:vocab + 1].cpu().numpy(), want, bound)
    assert bool((out[:, 0] == 5).all()) and bool((out[:, vocab + 1:] == 5).all())


# ---- verification of drafts ---------------------------------------------------------


def _verify_case(n, k, vocab, seed=1, sharp=3.0, near=0.5):
    r = _rng(n, k, vocab, seed)

    def softmax(z):
        e = np.exp(z - z.max(-1, keepdims=True))
        return (e / e.sum(-1, keepdims=True)).astype(np.float32)

    z = r.standard_normal((n, k + 1, vocab)) * sharp
    target = softmax(z)
    draft = softmax(z[:, :k] + r.standard_normal((n, k, vocab)) * near) if k else np.zeros((n, 0, vocab), np.float32)
    tok = np.zeros((n, k), np.int32)
    for i in range(n):
        for j in range(k):
            tok[i, j] = min(np.searchsorted(np.cumsum(draft[i, j].astype(np.float64)), r.random()), vocab - 1)
    return {"target": target, "draft": draft, "tok": tok, "n_draft": r.integers(0, k + 1, n).astype(np.int32),
            "ua": r.random((n, k)).astype(np.float32), "us": r.random(n).astype(np.float32)}


def _verify(sv, c, draft=True, n_draft=True):
    t, a = sv.verify_drafts_dev(_dev(c["target"]), _dev(c["tok"]), _dev(c["ua"]), _dev(c["us"]),
                                draft_probs=_dev(c["draft"]) if draft else None,
                                n_draft=_dev(c["n_draft"]) if n_draft else None)
    want_t, want_a = ref.verify(c["target"], c["draft"] if draft else None, c["tok"], c["n_draft"] if n_draft else None,
                                c["ua"], c["us"])
    assert np.array_equal(a.cpu().numpy(), want_a)
    assert np.array_equal(t.cpu().numpy(), want_t)
    return want_t, want_a


@pytest.mark.parametrize("n,k,vocab", [(1, 0, 1), (1, 1, 1), (1, 3, 7), (4, 4, 300), (9, 2, 2049), (2, 5, 32000),
                                       (40, 3, 1000), (3, 4, 151936), (1, 130, 50), (300, 1, 64), (1, 2, 151937), (2, 2, 8192),
                                       (1, 2, 8193), (2, 2, 32768), (2, 2, 32769), (90, 1, 33001)])
def test_verify_drafts_matches_its_definition(sv, n, k, vocab):
    c = _verify_case(n, k, vocab)
    for draft in (True, False):
        for n_draft in (True, False):
            _verify(sv, c, draft, n_draft)


def test_verify_drafts_all_and_none_accepted(sv):
    c = _verify_case(30, 4, 500)
    c["ua"][:] = 0.0
    _, acc = _verify(sv, c, n_draft=False)
    assert (acc == 4).all()
    c["ua"][:] = 1.0
    c["draft"] = np.maximum(c["draft"], c["target"][:, :4])  # never below the target: every product is refused
    _, acc = _verify(sv, c, n_draft=False)
    assert (acc == 0).all()


@pytest.mark.parametrize("vocab", [3000, 9000, 33003])
def test_verify_drafts_nothing_left_to_draw(sv, vocab):
    """p equal to q (nothing above it: the target's own row), p nowhere positive, a single positive value."""
    c = _verify_case(6, 2, vocab)
    c["ua"][:] = 1.0
    c["draft"][0] = c["target"][0, :2]
    c["draft"][1] = np.maximum(c["target"][1, :2], c["draft"][1])
    c["target"][2] = 0.0
    c["target"][3] = 0.0
    c["target"][3, :, vocab - 1] = 0.25
    c["target"][4] = 0.0
    c["target"][4, :, 0] = 1.0
    t, a = _verify(sv, c, n_draft=False)
    assert t[2, 0] == -1 and t[3, 0] == vocab - 1 and a[0] == 0
    _verify(sv, c, draft=False)


@pytest.mark.parametrize("vocab", [4097, 9000, 33003])
def test_verify_drafts_numbers_at_the_ends(sv, vocab):
    c = _verify_case(8, 1, vocab)
    c["us"][:] = [0.0, -1.0, np.nan, 1.0, 2.0, np.inf, 1.0 - 2.0 ** -24, -np.inf]
    c["target"][:, :, :100] = 0.0
    c["target"][:, :, -100:] = 0.0
    t, a = _verify(sv, c)
    _verify(sv, c, draft=False)
    drawn = t[np.arange(8), a]
    assert (drawn[[0, 1, 2, 7]] >= 100).all() and (drawn[[3, 4, 5]] < vocab - 100).all()


@pytest.mark.parametrize("vocab", [777, 9000, 33003])
def test_verify_drafts_strange_values(sv, vocab):
    """NaN, infinite and negative entries count as nothing; drafted tokens outside the vocabulary are refused; counts
    out of range are clamped."""
    c = _verify_case(12, 3, vocab)
    r = _rng(3)
    for bad in (np.nan, np.inf, -np.inf, -1.0):
        for name in ("target", "draft"):
            c[name][r.random(c[name].shape) < 0.05] = bad
    c["tok"][0, 0], c["tok"][1, 1], c["tok"][2, 0] = vocab, -1, 1 << 30
    c["ua"][3:5] = np.nan
    c["n_draft"][:] = [3, 3, 3, 3, 3, 99, -4, 0, 1, 2, 3, 3]
    for draft in (True, False):
        _, a = _verify(sv, c, draft)
        assert a[0] == 0 and a[1] <= 1 and a[2] == 0 and a[3] == 0 and a[6] == 0


def test_verify_drafts_same_token_in_every_place(sv):
    c = _verify_case(5, 4, 600)
    c["tok"][:] = 17
    _verify(sv, c)
    _verify(sv, c, draft=False)


def test_verify_drafts_beyond_32_bit_offsets(sv):
    """A target of 2^31 values and more: rows found at 64-bit offsets."""
    import torch

    n, k, vocab = 3, 4095, 190000
    target = torch.zeros((n, k + 1, vocab), device="cuda")
    assert target.numel() > 1 << 31
    tok = torch.full((n, k), 5, dtype=torch.int32, device="cuda")
    target[:, :, 5] = 1.0
    target[:, k] = 0.0
    target[0, k, 189999], target[1, k, 77777], target[2, k, 3] = 0.5, 0.5, 0.5
    u = torch.full((n, k), 0.5, device="cuda")
    t, a = sv.verify_drafts_dev(target, tok, u, torch.full((n,), 0.9, device="cuda"))
    assert a.tolist() == [k] * n
    assert t[:, k].tolist() == [189999, 77777, 3] and bool((t[:, :k] == 5).all())


def test_verify_drafts_distribution(sv):
    """The next token's share over many lanes of one row is the target's (acceptance and residual together): with N
    lanes a share's standard deviation is sqrt(p (1 - p) / N); the bound is six of them, the numbers fixed."""
    N, vocab = 20000, 12
    r = _rng(77)
    p = r.dirichlet(np.ones(vocab)).astype(np.float32)
    q = r.dirichlet(np.ones(vocab)).astype(np.float32)
    tok = np.searchsorted(np.cumsum(q.astype(np.float64)) / q.astype(np.float64).sum(), r.random(N)).astype(np.int32)[:, None]
    c = {"target": np.broadcast_to(p, (N, 2, vocab)).copy(), "draft": np.broadcast_to(q, (N, 1, vocab)).copy(), "tok": tok,
         "n_draft": np.ones(N, np.int32), "ua": r.random((N, 1)).astype(np.float32), "us": r.random(N).astype(np.float32)}
    t, _ = sv.verify_drafts_dev(_dev(c["target"]), _dev(c["tok"]), _dev(c["ua"]), _dev(c["us"]), draft_probs=_dev(c["draft"]))
    share = np.bincount(t.cpu().numpy()[:, 0], minlength=vocab) / N
    pn = p.astype(np.float64) / p.astype(np.float64).sum()
    assert (np.abs(share - pn) <= 6 * np.sqrt(pn * (1 - pn) / N)).all()


# ---- the calls among others --------------------------------------------------------


def _head(s, o):
    """Stands for the output head: each logit one output value times a weight."""
    return o.reshape(-1, 512)[:, s["at"]] * s["head"]


def _step(sv, s):
    """One verification step's operators in the order a server runs them, each on the one before's output."""
    q = sv.lora_dev(s["x"], s["a"], s["b"], s["scale"], s["ids"], base=s["base"])
    o = sv.prefix_attn_dev(q.view(s["n"], s["nq"], 8, 64), s["kp"], s["vp"], s["ko"], s["vo"], s["own_len"], 0.125,
                           q_len=s["q_len"])
    logits = _head(s, o)
    p = sv.token_probs_dev(logits, s["temp"])
    t, a = sv.verify_drafts_dev(p.view(s["n"], s["nq"], -1), s["tok"], s["ua"], s["us"], n_draft=s["q_len"] - 1)
    return q, o, p, t, a


def _step_inputs(n=6, nq=4, vocab=3001, rank=16, seed=1):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)

    def f(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def i(hi, *shape):
        return torch.randint(0, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    return {"n": n, "nq": nq, "x": f(n * nq, 256), "base": f(n * nq, 512), "a": (f(5, rank, 256) / 16).half(),
            "b": (f(5, 512, rank) / rank ** 0.5).half(), "scale": torch.ones(5, device="cuda"), "ids": i(6, n * nq) - 1,
            "kp": f(300, 2, 64).half(), "vp": f(300, 2, 64).half(), "ko": f(n, 50, 2, 64).half(), "vo": f(n, 50, 2, 64).half(),
            "own_len": i(47, n) + 4, "q_len": i(nq, n) + 1, "head": f(vocab) * 9, "at": i(512, vocab).long(), "temp": torch.full((n * nq,), 0.7, device="cuda"),
            "tok": i(vocab, n, nq - 1), "ua": torch.rand((n, nq - 1), generator=g, device="cuda") * 1e-4,
            "us": torch.rand((n,), generator=g, device="cuda")}


FORMS = pytest.mark.parametrize("vocab,rank", [(3001, 16), (33001, 128)])  # one launch a call, and two


@FORMS
def test_a_step_of_all_operators(sv, vocab, rank):
    """The four together, each stage held to its definition on the stage before's output."""
    s = _step_inputs(vocab=vocab, rank=rank)
    q, o, p, t, a = _step(sv, s)
    h = {k: (v.float() if v.is_floating_point() else v).cpu().numpy() for k, v in s.items() if hasattr(v, "cpu")}
    want, bound = ref.lora(h["x"], h["a"], h["b"], h["scale"], h["ids"], h["base"])
    _within(q.cpu().numpy(), want, bound, "lora")
    want, bound = ref.prefix_attn(q.cpu().numpy().reshape(6, 4, 8, 64), h["kp"], h["vp"], h["ko"], h["vo"], h["own_len"],
                                  h["q_len"], 0.125)
    _within(o.cpu().numpy(), want, bound, "attention")
    logits = _head(s, o).cpu().numpy()
    want, bound = ref.token_probs(logits, h["temp"])
    _within(p.cpu().numpy(), want, bound, "probabilities")
    want_t, want_a = ref.verify(p.cpu().numpy().reshape(6, 4, -1), None, h["tok"], h["q_len"] - 1, h["ua"], h["us"])
    assert np.array_equal(t.cpu().numpy(), want_t) and np.array_equal(a.cpu().numpy(), want_a)


def test_beside_a_quantized_projection(sv):
    """Adapters in place over matvec_dev's output, for lanes of a batch: the projection's own bits below them."""
    import torch

    from loom_amd import Q4_K, backend as be

    n, rows, cols = 9, 512, 1024
    w = be.repack_dev(Q4_K, be.synth_ggml_dev(Q4_K, rows, cols, 1, 3, 0.02), rows, cols, 1)
    t = _lora_case(n, rows, cols, 16, 4, "f16")
    out = torch.empty(n, rows, device="cuda")
    be.matvec_dev(Q4_K, out, w, t["x"], n, rows, cols)
    t["base"] = out.clone()
    sv.lora_dev(t["x"], t["a"], t["b"], t["scale"], t["ids"], base=out, out=out)
    want, bound = _lora_ref(t)
    _within(out.cpu().numpy(), want, bound)
    assert bool((out[t["ids"] < 0] == t["base"][t["ids"] < 0]).all())


@FORMS
def test_repeated_calls_give_the_same_bits(sv, vocab, rank):
    s = _step_inputs(n=33, nq=3, vocab=vocab, rank=rank)
    first = _step(sv, s)
    for _ in range(3):
        for x, y in zip(first, _step(sv, s)):
            assert bool((x == y).all())


@FORMS
def test_captured_steps_replay(sv, vocab, rank):
    """Two captured graphs of the step, replayed in turn on inputs that change in place, with eager calls and other
    allocations between the replays: each replay equals the eager result."""
    import torch

    form = {"vocab": vocab, "rank": rank}
    a, b = _step_inputs(**form), _step_inputs(n=3, nq=2, seed=9, **form)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in (a, b):
            _step(sv, s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(sv, s)
        graphs.append((g, out, s))
    fresh = ([_step_inputs(seed=20 + k, **form) for k in range(3)],
             [_step_inputs(n=3, nq=2, seed=30 + k, **form) for k in range(3)])
    for k in range(3):
        for (g, out, s), new in zip(graphs, fresh):
            for key in ("x", "ids", "own_len", "q_len", "us", "ua", "tok"):
                s[key].copy_(new[k][key])
            want = [t.clone() for t in _step(sv, s)]
            torch.empty(1 << 20, device="cuda").fill_(float("nan"))
            for t in out:
                t.fill_(-7)
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, want):
                assert bool((x == y).all()), k


@FORMS
def test_steps_on_two_streams(sv, vocab, rank):
    import torch

    sets = [_step_inputs(n=20, nq=3, vocab=vocab, rank=rank, seed=k) for k in (1, 2)]
    want = [_step(sv, s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(_step(sv, sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            for x, y in zip(out, want[k]):
                assert bool((x == y).all())


@FORMS
def test_calls_from_two_threads(sv, vocab, rank):
    import threading

    import torch

    sets = [_step_inputs(n=20, nq=3, vocab=vocab, rank=rank, seed=k) for k in (3, 4)]
    want = [_step(sv, s) for s in sets]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[k] = _step(sv, sets[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors
    for k in range(2):
        for x, y in zip(got[k], want[k]):
            assert bool((x == y).all())


def test_empty_batches(sv):
    import torch

    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    i32, h = torch.int32, torch.float16
    assert sv.prefix_attn_dev(z(0, 1, 4, 64), z(5, 2, 64, dt=h), z(5, 2, 64, dt=h), None, None, None, 1.0).shape == (0, 1, 4, 64)
    assert sv.prefix_attn_dev(z(2, 0, 4, 64), z(5, 2, 64, dt=h), z(5, 2, 64, dt=h), None, None, None, 1.0).shape == (2, 0, 4, 64)
    assert sv.lora_dev(z(0, 8), z(1, 2, 8), z(1, 3, 2), z(1), z(0, dt=i32)).shape == (0, 3)
    assert sv.token_probs_dev(z(0, 100)).shape == (0, 100)
    t, a = sv.verify_drafts_dev(z(0, 3, 9), z(0, 2, dt=i32), z(0, 2), z(0))
    assert t.shape == (0, 3) and a.shape == (0,)
