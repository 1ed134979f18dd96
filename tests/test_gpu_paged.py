"""The operators around a paged cache on the device against their definitions
in 64 bits (paged_ref.py, elementwise error bounds derived there), at the
sizes, layouts, masks and values where they can go wrong, and together."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sv():
    import loom_amd
    from loom_amd import serving

    loom_amd.init(0)
    return serving


def _rng(*key):
    return np.random.default_rng([int(k) for k in key])


def _dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _half(a, kind):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch.float16 if kind == "f16" else torch.bfloat16)


def _np(t):
    return t.double().cpu().numpy()


def _within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    ok = ~np.isnan(want)
    assert np.isfinite(got[ok]).all(), what
    off = np.abs(got[ok] - want[ok]) - bound[ok]
    assert off.size == 0 or off.max() <= 0, f"{what}: {off.max()} over the bound, {np.abs(got[ok] - want[ok]).max()} off"


# ---- norms and rotation -----------------------------------------------------------


def _rope_case(n, H, KV, hd, rot, far=5000, norm=True, seed=0):
    r = _rng(n, H, KV, hd, rot, seed)
    c = {"q": (r.standard_normal((n, H, hd)) * 2).astype(np.float32), "k": r.standard_normal((n, KV, hd)).astype(np.float32),
         "pos": r.integers(0, far, n).astype(np.int32),
         "freqs": 1.0 / 10000.0 ** (np.arange(0, rot, 2) / max(rot, 1)) if rot else None,
         "q_norm": (1 + r.standard_normal(hd) * 0.1).astype(np.float32) if norm else None,
         "k_norm": (1 + r.standard_normal(hd) * 0.1).astype(np.float32) if norm else None}
    return c


def _opt(a):
    return None if a is None else _dev(a)


ROPE = [
    # n, heads, key heads, head size, rotated
    (1, 1, 1, 8, 8), (1, 32, 4, 128, 128), (5, 6, 6, 48, 32), (3, 2, 1, 64, 64), (7, 3, 2, 40, 20), (2, 4, 4, 256, 256),
    (33, 5, 1, 96, 96), (3, 8, 2, 200, 100), (9, 7, 3, 16, 2), (2, 71, 1, 64, 0), (300, 32, 4, 128, 64), (1000, 9, 2, 80, 80),
    (611, 14, 3, 24, 8), (257, 40, 8, 256, 128), (4, 3, 1, 120, 118),
]


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("shape", ROPE, ids=lambda s: "x".join(map(str, s)))
def test_qk_norm_rope_matches_its_definition(sv, shape, inter):
    for norm in (True, False):
        c = _rope_case(*shape, norm=norm)
        got = sv.qk_norm_rope_dev(_dev(c["q"]), _dev(c["k"]), _dev(c["pos"]), _opt(c["freqs"]), q_norm=_opt(c["q_norm"]),
                                  k_norm=_opt(c["k_norm"]), eps=1e-5, interleaved=inter)
        for name, g in zip("qk", got):
            _within(_np(g), *ref.norm_rope(c[name], c["pos"], c["freqs"], c[name + "_norm"], 1e-5, inter), (name, norm))


def test_qk_norm_rope_at_far_positions(sv):
    c = _rope_case(64, 4, 2, 128, 128)
    c["pos"] = _rng(3).integers(2 ** 30, 2 ** 31 - 1, 64).astype(np.int32)
    c["pos"][:3] = 0, 2 ** 31 - 1, 2 ** 24 + 1
    q, k = sv.qk_norm_rope_dev(_dev(c["q"]), _dev(c["k"]), _dev(c["pos"]), _dev(c["freqs"]))
    # the definition's own angles are off by 2^-53 of two billion: 2e-7, four roundings of 1
    for name, g in (("q", q), ("k", k)):
        want, bound = ref.norm_rope(c[name], c["pos"], c["freqs"], None, 0, False)
        _within(_np(g), want, bound * 2)


def test_qk_norm_rope_in_place_and_strided(sv):
    import torch

    for shape, inter in (((40, 8, 2, 64, 64), False), ((700, 16, 4, 128, 96), True), ((6, 4, 2, 40, 20), False)):
        n, H, KV, hd, rot = shape
        c = _rope_case(*shape)
        args = (_dev(c["pos"]), _dev(c["freqs"]))
        norms = {"q_norm": _dev(c["q_norm"]), "k_norm": _dev(c["k_norm"]), "interleaved": inter}
        want = sv.qk_norm_rope_dev(_dev(c["q"]), _dev(c["k"]), *args, **norms)
        # column groups of one buffer, one value past an aligned start, in place
        buf = torch.full((n, 3 + (H + KV) * hd + 5), 7.0, device="cuda")
        q, k = buf[:, 3:3 + H * hd].unflatten(1, (H, hd)), buf[:, 3 + H * hd:3 + (H + KV) * hd].unflatten(1, (KV, hd))
        q.copy_(_dev(c["q"])), k.copy_(_dev(c["k"]))
        got = sv.qk_norm_rope_dev(q, k, *args, **norms, q_out=q, k_out=k)
        assert got[0] is q and got[1] is k
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert (buf[:, :3] == 7).all() and (buf[:, 3 + (H + KV) * hd:] == 7).all()
        alone = sv.qk_norm_rope_dev(_dev(c["q"]), None, *args, **norms)
        assert torch.equal(alone[0], want[0]) and alone[1] is None


def test_qk_norm_rope_leaves_padding(sv):
    import torch

    c = _rope_case(50, 8, 2, 64, 64)
    c["pos"][::3] = -1
    c["pos"][7] = -2 ** 31
    q, k = torch.full((50, 8, 64), 5.0, device="cuda"), torch.full((50, 2, 64), 5.0, device="cuda")
    sv.qk_norm_rope_dev(_dev(c["q"]), _dev(c["k"]), _dev(c["pos"]), _dev(c["freqs"]), q_out=q, k_out=k)
    for name, g in (("q", q), ("k", k)):
        want, bound = ref.norm_rope(c[name], c["pos"], c["freqs"], None, 0, False)
        _within(_np(g), want, bound)
        assert (g[_dev(c["pos"] < 0)] == 5).all()


def test_qk_norm_rope_of_nothing_and_of_no_number(sv):
    import torch

    c = _rope_case(4, 2, 1, 64, 64)
    c["q"][1] = 0.0
    c["q"][2, 0, 5] = np.nan
    c["q"][2, 1, 5] = np.inf
    args = (_dev(c["pos"]), _dev(c["freqs"]))
    q, _ = sv.qk_norm_rope_dev(_dev(c["q"]), None, *args, q_norm=_dev(c["q_norm"]))
    assert (q[1] == 0).all() and q[2, 0].isnan().all() and torch.isfinite(q[[0, 3]]).all()
    q, _ = sv.qk_norm_rope_dev(_dev(c["q"]), None, *args)
    assert q[2, 0].isnan().nonzero().flatten().tolist() == [5, 37]
    e = torch.empty(0, 2, 64, device="cuda")
    assert sv.qk_norm_rope_dev(e, None, args[0][:0], args[1])[0].shape == (0, 2, 64)


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("hd,rot", [(64, 20), (64, 2), (24, 12), (128, 126), (256, 250), (64, 32)])
def test_what_is_not_rotated_stays_as_it_is(sv, hd, rot, inter):
    """Infinities, NaN and -0 right behind the rotated values leave their neighbours alone, in q, k and the pages."""
    import torch

    n, H, KV, ps = 6, 3, 2, 4
    c = _rope_case(n, H, KV, hd, rot, norm=False)
    c["pos"] = np.arange(n, dtype=np.int32)
    for x in (c["q"], c["k"]):
        for t, odd in enumerate((np.inf, -np.inf, np.nan, -0.0)):
            for h in range(x.shape[1]):
                x[t, h, rot + (h + t) % min(6, hd - rot)] = odd  # in the same four pairs as the last rotated ones, and behind
        x[4, :, rot:] = -0.0
    q0, k0 = _dev(c["q"]), _dev(c["k"])
    q, k = sv.qk_norm_rope_dev(q0, k0, _dev(c["pos"]), _dev(c["freqs"]), interleaved=inter)
    for name, x, got in (("q", q0, q), ("k", k0, k)):
        assert torch.equal(got[..., rot:].contiguous().view(torch.int32), x[..., rot:].contiguous().view(torch.int32)), name
        part = {"x": c[name][..., :rot], "pos": c["pos"], "freqs": c["freqs"], "w": None, "eps": 0, "interleaved": inter}
        _within(_np(got[..., :rot]), *ref.norm_rope(**part), name)
    for kind, dt in (("f16", torch.float16), ("bf16", torch.bfloat16)):
        kp, vp = _cache(2, ps, KV, hd, kind)
        sv.paged_append_dev(k0, k0, kp, vp, _dev(np.array([[1, 0]], np.int32)), _dev(c["pos"]), freqs=_dev(c["freqs"]),
                            lanes=_dev(np.zeros(n, np.int32)), interleaved=inter)
        for t in range(n):
            got, want = kp[1 - t // ps, t % ps, :, rot:].float(), k0[t, :, rot:].to(dt).float()
            assert torch.equal(got.isnan(), want.isnan())
            assert ((got == want) & (got.signbit() == want.signbit()) | want.isnan()).all(), (kind, t)


# ---- into the pages ---------------------------------------------------------------


def _cache(n_pages, ps, KV, hd, kind, layout="rows", seed=5):
    """Two pools of random rows; `heads`: a page's rows lie head by head, `pair`: keys and values share one buffer."""
    import torch

    r = _rng(n_pages, ps, KV, hd, seed)
    x = _half(r.standard_normal((2, n_pages, ps, KV, hd)), kind).cuda()
    if layout == "heads":
        x = x.transpose(2, 3).contiguous().transpose(2, 3)
    if layout == "pair":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    return x[0], x[1]


def _table(lens, ps, n_pages, width=None, seed=0):
    """A table over pages in any order; entries past a lane's rows are -1."""
    used = [-(-int(x) // ps) for x in lens]
    order = _rng(seed, *used).permutation(n_pages)
    t = np.full((len(lens), width or max(max(used), 1)), -1, np.int32)
    at = 0
    for i, u in enumerate(used):
        t[i, :u] = order[at:at + u]
        at += u
    return t


APPEND = [
    # lanes, tokens a lane, heads, key heads, head size, page size, kind, layout
    (1, 1, 32, 4, 128, 16, "f16", "rows"),
    (3, 5, 6, 6, 48, 7, "bf16", "heads"),
    (33, 1, 8, 2, 64, 1, "f16", "pair"),
    (2, 300, 16, 2, 128, 64, "bf16", "rows"),
    (5, 17, 3, 1, 256, 24, "f16", "heads"),
    (4, 40, 5, 5, 40, 128, "bf16", "pair"),
]


@pytest.mark.parametrize("shape", APPEND, ids=lambda s: "x".join(map(str, s)))
def test_paged_append_matches_its_definition(sv, shape):
    import torch

    n, new, H, KV, hd, ps, kind, layout = shape
    rot = {48: 32, 40: 20}.get(hd, hd)
    T = n * new
    c = _rope_case(T, H, KV, hd, rot)
    v = _rng(9).standard_normal((T, KV, hd)).astype(np.float32)
    lens = [new + 11 * i for i in range(n)]
    n_pages = sum(-(-x // ps) for x in lens) + 3
    table = _table(lens, ps, n_pages)
    order = _rng(T).permutation(T)  # tokens in any order
    lanes = np.repeat(np.arange(n), new).astype(np.int32)[order]
    pos = np.concatenate([np.arange(x - new, x) for x in lens]).astype(np.int32)[order]
    if T > 3:
        pos[1] = -1
    for inter in (False, True):
        kp, vp = _cache(n_pages, ps, KV, hd, kind, layout)
        k0, v0 = _np(kp), _np(vp)
        q = sv.paged_append_dev(_dev(c["k"]), _dev(v), kp, vp, _dev(table), _dev(pos), lanes=_dev(lanes), freqs=_dev(c["freqs"]),
                                k_norm=_dev(c["k_norm"]), q=_dev(c["q"]), q_norm=_dev(c["q_norm"]), interleaved=inter)
        _within(_np(q), *ref.norm_rope(c["q"], pos, c["freqs"], c["q_norm"], 1e-6, inter), "q")
        want, bound = ref.norm_rope(c["k"], pos, c["freqs"], c["k_norm"], 1e-6, inter)
        bk, bv = np.zeros(k0.shape), np.zeros(v0.shape)
        for t, at in enumerate(ref.slots(table, n_pages, ps, pos, lanes)):
            if at:
                k0[at], bk[at] = want[t], ref.rounded(want[t], bound[t], kind)
                v0[at] = _np(_half(v[t], kind))  # exactly
        _within(_np(kp), k0, bk, "keys")
        assert (_np(vp) == v0).all()
        # without queries, and with the lanes as they come: the same rows
        k2, v2 = _cache(n_pages, ps, KV, hd, kind, layout)
        assert sv.paged_append_dev(_dev(c["k"]), _dev(v), k2, v2, _dev(table), _dev(pos), lanes=_dev(lanes),
                                   freqs=_dev(c["freqs"]), k_norm=_dev(c["k_norm"]), interleaved=inter) is None
        assert torch.equal(k2, kp) and torch.equal(v2, vp)


def test_paged_append_drops_what_has_no_page(sv):
    """Padding, lanes outside the table, positions past it, entries outside the pool: nothing is written."""
    import torch

    kp, vp = _cache(6, 8, 2, 64, "f16")
    k0, v0 = kp.clone(), vp.clone()
    table = np.array([[0, 1, -1], [6, 2 ** 31 - 1, 2], [3, -2 ** 31, 4]], np.int32)
    lanes = np.array([0, 0, 0, 1, 1, 1, 2, -1, 3, 2 ** 31 - 1, 2], np.int32)
    pos = np.array([-1, 24, 17, 0, 8, 16, 8, 0, 0, 0, 2 ** 31 - 1], np.int32)
    T = len(pos)
    r = _rng(4)
    k, v, q = (_dev(r.standard_normal((T, h, 64)).astype(np.float32)) for h in (2, 2, 4))
    out = torch.full((T, 4, 64), 3.0, device="cuda")
    sv.paged_append_dev(k, v, kp, vp, _dev(table), _dev(pos), lanes=_dev(lanes), q=q, q_out=out)
    kept = [i for i in range(T) if i != 5]
    assert ref.slots(table, 6, 8, pos, lanes) == [(2, 0) if i == 5 else None for i in range(T)]
    k0[2, 0], v0[2, 0] = k[5].half(), v[5].half()
    assert torch.equal(kp, k0) and torch.equal(vp, v0) and kept
    assert (out[0] == 3).all() and torch.equal(out[1:], q[1:])  # queries of all but padding


def test_paged_append_rounds_to_the_nearest(sv):
    """Ties to even, f16's subnormals, overflow to infinity, NaN: as torch rounds."""
    import torch

    x = np.float32([1 + 2 ** -11, 1 + 3 * 2 ** -11, 65519.9, 65520.0, 1e30, 2 ** -25, 1.5 * 2 ** -24, -0.0, np.nan, np.inf,
                    1 + 2 ** -8, 1 + 3 * 2 ** -8, 3.4e38, 1e-40, -65520.0, 2 ** -24])
    for kind, dt in (("f16", torch.float16), ("bf16", torch.bfloat16)):
        kp, vp = (torch.zeros(1, 1, 2, 8, dtype=dt, device="cuda") for _ in range(2))
        k = _dev(x.reshape(1, 2, 8))
        sv.paged_append_dev(k, k, kp, vp, _dev(np.zeros((1, 1), np.int32)), _dev(np.zeros(1, np.int32)))
        want = k.to(dt).view(torch.int16)[0]
        for got in (kp, vp):
            assert torch.equal(got[0, 0].isnan(), k[0].isnan())
            assert ((got[0, 0].view(torch.int16) == want) | k[0].isnan()).all()


# ---- attention over pages ---------------------------------------------------------


ATTN = [
    # heads, key heads, head size, page size, lens, kind, layout
    (1, 1, 8, 1, [1], "f16", "rows"),
    (32, 4, 128, 16, [256], "f16", "rows"),
    (32, 4, 128, 16, [0, 1, 31, 32, 33, 127, 128, 129, 500], "f16", "heads"),
    (6, 6, 48, 24, [5, 0, 333, 64, 65, 63], "bf16", "rows"),
    (16, 2, 64, 7, [700, 3, 129], "bf16", "pair"),
    (8, 2, 256, 64, [1, 300, 31, 32, 97], "f16", "rows"),
    (8, 2, 256, 5, [200, 33], "bf16", "heads"),
    (40, 2, 80, 128, [260, 1000, 2], "f16", "rows"),      # a group of 20: two blocks of heads
    (71, 1, 64, 32, [90, 400], "bf16", "rows"),           # more heads than four blocks
    (28, 4, 128, 100, [2500, 10, 0, 777], "bf16", "pair"),
    (24, 8, 96, 16, [1500, 64], "f16", "pair"),
    (2, 1, 128, 256, [9000], "f16", "rows"),
    (4, 4, 200, 48, [50, 4000], "f16", "rows"),
    (16, 16, 16, 3, list(range(40)), "bf16", "rows"),
]


def _attn_case(H, KV, hd, ps, lens, kind, layout, seed=0, spare=2, width=None):
    r = _rng(H, KV, hd, ps, *lens, seed)
    n_pages = sum(-(-x // ps) for x in lens) + spare
    kp, vp = _cache(n_pages, ps, KV, hd, kind, layout)
    return {"q": r.standard_normal((len(lens), H, hd)).astype(np.float32), "kp": kp, "vp": vp,
            "table": _table(lens, ps, n_pages, width), "lens": np.array(lens, np.int32), "scale": hd ** -0.5, "window": 0}


def _attn(sv, c, out=None):
    return sv.paged_attn_dev(_dev(c["q"]), c["kp"], c["vp"], _dev(c["table"]), _dev(c["lens"]), c["scale"], window=c["window"],
                             out=out)


def _attn_ref(c):
    return ref.attn(c["q"], _np(c["kp"]), _np(c["vp"]), c["table"], c["lens"], c["scale"], c["window"])


@pytest.mark.parametrize("shape", ATTN, ids=lambda s: "x".join(str(x) if not isinstance(x, list) else f"{len(x)}of{max(x)}" for x in s))
def test_paged_attn_matches_its_definition(sv, shape):
    c = _attn_case(*shape)
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound)
    assert (got[c["lens"] == 0] == 0).all()
    for window in (1, 30, 130):
        c["window"] = window
        _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), window)


def test_paged_attn_splits_long_lanes(sv):
    """Few lanes of very unequal lengths: one is cut into many ranges, some hold a few rows."""
    for lens, kv, H, hd, kind in (([40000, 1, 17, 0, 300], 2, 16, 64, "f16"), ([33333], 1, 3, 128, "bf16"),
                                  ([20000, 20000, 5], 4, 4, 32, "f16"), ([12345, 7], 1, 40, 128, "f16"),
                                  ([6000, 1], 2, 4, 256, "bf16")):
        c = _attn_case(H, kv, hd, 16, lens, kind, "rows")
        _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), lens)


@pytest.mark.parametrize("n", [300, 1100])
def test_paged_attn_many_lanes(sv, n):
    r = _rng(n)
    c = _attn_case(4, 2, 32, 8, [int(x) for x in r.integers(0, 60, n)], "f16", "rows")
    c["lens"][n // 2:n // 2 + 20] = 0
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound)
    assert (got[c["lens"] == 0] == 0).all()


@pytest.mark.parametrize("shape", [
    # heads, key heads, head size, lanes, longest: in more items than run at a time, in fewer, with one long lane
    (8, 4, 32, 200, 1300, "f16"), (4, 4, 16, 130, 700, "bf16"), (3, 1, 128, 90, 1100, "f16"), (20, 1, 256, 70, 600, "bf16"),
    (2, 2, 64, 65, 900, "f16"),
], ids=lambda s: "x".join(map(str, s)))
def test_paged_attn_many_lanes_are_cut(sv, shape):
    H, KV, hd, n, longest, kind = shape
    r = _rng(n, longest)
    lens = [int(x) for x in r.integers(0, longest, n)]
    lens[3:9] = [0] * 6
    lens[n - 2] = 20 * longest
    c = _attn_case(H, KV, hd, 16, lens, kind, "rows")
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound)
    assert (got[c["lens"] == 0] == 0).all()
    c["window"] = 300
    _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), "window")


def test_paged_attn_thousands_of_lanes_are_cut(sv):
    """More lanes than a wave has threads, many times over, most of them short; a page each that holds more than is left
    whole."""
    n = 2500
    r = _rng(n)
    lens = r.integers(0, 30, n)
    lens[r.permutation(n)[:12]] = r.integers(300, 601, 12)
    kp, vp = _cache(n, 600, 1, 8, "f16")
    c = {"q": r.standard_normal((n, 2, 8)).astype(np.float32), "kp": kp, "vp": vp,
         "table": r.permutation(n).astype(np.int32)[:, None], "lens": lens.astype(np.int32), "scale": 0.5, "window": 0}
    want, bound = _attn_ref(c)
    got = _attn(sv, c).cpu().numpy()
    _within(got, want, bound)
    assert (got[c["lens"] == 0] == 0).all()


def test_paged_attn_of_a_decoders_caches(sv):
    """Contiguous caches are pages of one lane each: [n, layers, ctx, kvd] at a layer."""
    import torch

    n, layers, ctx, KV, hd = 3, 4, 700, 2, 64
    r = _rng(3)
    cache = torch.from_numpy(r.standard_normal((2, n, layers, ctx, KV * hd)).astype(np.float32)).half().cuda()
    for layer in (0, 3):
        kp, vp = (x[:, layer].unflatten(-1, (KV, hd)) for x in cache)
        c = {"q": r.standard_normal((n, 8, hd)).astype(np.float32), "kp": kp, "vp": vp,
             "table": np.arange(n, dtype=np.int32)[:, None], "lens": np.array([700, 1, 333], np.int32), "scale": hd ** -0.5,
             "window": 0}
        _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), layer)


def test_paged_attn_empty_batch_in_a_wide_table(sv):
    c = _attn_case(8, 2, 64, 16, [40, 0, 3], "f16", "rows", width=400)
    for lens in ([0, 0, 0], [0, 0, 1], [40, 0, 3]):
        c["lens"] = np.array(lens, np.int32)
        want, bound = _attn_ref(c)
        got = _attn(sv, c).cpu().numpy()
        _within(got, want, bound, lens)
        assert (got[c["lens"] == 0] == 0).all()


def test_paged_attn_lengths_past_the_table(sv):
    """A length is clamped into what the table can hold; a table wider than the lengths changes nothing."""
    import torch

    c = _attn_case(8, 2, 64, 16, [64, 64, 48], "f16", "rows")
    c["table"][2, 3] = 0
    want = _attn(sv, c)
    for extra in ((2 ** 31 - 1, 65, 48), (64, 64, 48)):
        c["lens"] = np.array(extra, np.int32)
        assert torch.equal(_attn(sv, c), want)
    c["lens"] = np.array([-1, -2 ** 31, 48], np.int32)
    got = _attn(sv, c)
    assert (got[:2] == 0).all() and torch.equal(got[2], want[2])
    c = _attn_case(8, 2, 64, 16, [64, 64, 48], "f16", "rows")
    wide = np.concatenate([c["table"], np.full((3, 5000), -1, np.int32)], 1)
    got = _attn(sv, {**c, "table": wide}).cpu().numpy()
    _within(got, *_attn_ref(c), "wide")


def test_paged_attn_pages_that_are_not_there(sv):
    """Entries outside the pool are not seen, wherever they stand; a lane of such alone sees nothing."""
    c = _attn_case(8, 2, 128, 16, [700, 200, 33, 512], "f16", "rows")
    n_pages = c["kp"].shape[0]
    c["table"][0, :20] = -1                       # given back
    c["table"][1, [0, 5, 12]] = n_pages, 2 ** 31 - 1, -2 ** 31
    c["table"][2, :] = -7
    c["table"][3, 31] = n_pages
    for window in (0, 100):
        c["window"] = window
        want, bound = _attn_ref(c)
        got = _attn(sv, c).cpu().numpy()
        _within(got, want, bound, window)
        assert (got[2] == 0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_paged_attn_rows_not_seen_hold_anything(sv, kind):
    """NaN and infinities in the rest of a last page, before a window and in pages of no lane."""
    import torch

    c = _attn_case(8, 2, 64, 24, [100, 31, 250, 3], kind, "rows", spare=5)
    for window in (0, 40):
        c["window"] = window
        want, bound = _attn_ref(c)
        seen = torch.zeros(c["kp"].shape[:2], dtype=torch.bool)
        for i, x in enumerate(c["lens"]):
            t = np.arange(max(0, x - window) if window else 0, x)
            seen[c["table"][i][t // 24], t % 24] = True
        for bad in (float("nan"), float("inf"), -float("inf")):
            dirty = {**c, "kp": c["kp"].clone(), "vp": c["vp"].clone()}
            dirty["kp"][~seen], dirty["vp"][~seen] = bad, bad
            _within(_attn(sv, dirty).cpu().numpy(), want, bound, (window, bad))


def test_paged_attn_no_numbers_that_are_seen(sv):
    import torch

    c = _attn_case(8, 2, 64, 16, [100, 100, 100, 100], "f16", "rows")
    clean = _attn(sv, c)
    page = lambda i, t: (int(c["table"][i, t // 16]), t % 16)
    c["vp"][page(0, 50)][0, 3] = float("nan")
    c["vp"][page(1, 99)][1, 7] = float("inf")
    c["kp"][page(2, 0)][0, 0] = float("nan")
    got = _attn(sv, c)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :4, 3] = bad[1, 4:, 7] = bad[2, :4] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("scale", [-0.25, 0.0, 30.0, 1e-30])
def test_paged_attn_scales(sv, scale):
    for kind in ("f16", "bf16"):
        c = _attn_case(8, 2, 64, 16, [400, 33], kind, "rows")
        c["scale"] = scale
        _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), (scale, kind))


@pytest.mark.parametrize("size", [1e-30, 1e-3, 300.0, 1e20])
def test_paged_attn_queries_of_any_size(sv, size):
    """The scores stay ordinary: the scale takes the query's size out."""
    for kind in ("f16", "bf16"):
        c = _attn_case(4, 1, 128, 16, [400, 33], kind, "rows")
        c["q"] = (c["q"] * size).astype(np.float32)
        c["scale"] = 0.1 / size
        _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), (size, kind))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("size", [3e6, 1e9, 1e30])
def test_paged_attn_of_one_row_that_outweighs_all(sv, kind, size):
    """Scores of millions and more: the row of the largest alone, its value exactly."""
    c = _attn_case(4, 2, 64, 16, [700, 90], kind, "rows")
    want = _np(_attn(sv, c)) * 0
    r = _rng(5)
    for i, n in enumerate((700, 90)):
        for h in range(4):
            k = _np(c["kp"])[c["table"][i][np.arange(n) // 16], np.arange(n) % 16, h // 2]
            best = int(r.integers(0, n))
            c["q"][i, h] = k[best] * size  # |k|^2 against k . k': the largest by some units, times size
            s = k @ k[best]
            assert s[best] - np.delete(s, best).max() > 0.5
            want[i, h] = _np(c["vp"])[c["table"][i][best // 16], best % 16, h // 2]
    c["scale"] = 1.0
    assert (_np(_attn(sv, c)) == want).all()


BIG = [
    # heads, key heads, head size, page size, lens: whole lanes, and lanes that are cut
    (8, 2, 64, 16, [4, 1, 100, 3, 64]), (8, 2, 256, 16, [2, 90, 0, 127]), (4, 1, 128, 16, [5000, 4, 700]),
    (2, 1, 256, 32, [3000, 2]), (20, 1, 48, 16, [40000, 65, 4096]),
]


@pytest.mark.parametrize("kind,big", [("bf16", 3.38e38), ("f16", 65504.0)])
@pytest.mark.parametrize("shape", BIG, ids=lambda s: "x".join(map(str, s[:4])) + f"x{max(s[4])}")
def test_paged_attn_values_at_the_end_of_the_range(sv, shape, kind, big):
    """A weighted mean is no larger than its largest value: finite values have finite results, whatever their sums."""
    c = _attn_case(*shape, kind, "rows")
    r = _rng(5, *shape[:4])
    signs = [np.ones(c["vp"].shape), -np.ones(c["vp"].shape), r.choice([-1.0, 1.0], c["vp"].shape)]
    for q in (0.0, 1.0):  # equal weights, others
        c["q"] = c["q"] * np.float32(q)
        for s in signs + [r.uniform(-1, 1, c["vp"].shape)]:
            c["vp"].copy_(_half(s * big, kind))
            _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c), q)
        c["q"] = r.standard_normal(c["q"].shape).astype(np.float32)
    c["vp"].copy_(_half(signs[0] * big, kind))
    c["q"][:] = 0
    top = _np(c["vp"][0, 0, 0, 0])
    got = _np(_attn(sv, c))[c["lens"] > 0]
    # the sum of T weights of 2^-k, the products of the value, the quotient: off by the sums' roundings, T EPS at most
    assert (np.abs(got / top - 1) <= (max(shape[4]) + 40) * 2.0 ** -24).all()


@pytest.mark.parametrize("lens", [[33, 2, 200], [9000, 700]], ids=["whole", "cut"])
def test_paged_attn_weights_far_below_the_largest(sv, lens):
    """One row of nearly all the weight and the value 0; the result is the others' share, 2^-90 of their values."""
    hd = 64
    c = _attn_case(2, 1, hd, 16, lens, "bf16", "rows")
    c["kp"][:], c["vp"][:] = 0, float(2.0 ** 100)
    for i, n in enumerate(lens):
        t = n // 2
        c["kp"][int(c["table"][i, t // 16]), t % 16, 0, 3] = 1.0
        c["vp"][int(c["table"][i, t // 16]), t % 16] = 0
    c["q"][:] = 0
    c["q"][:, :, 3] = 1.0
    c["scale"] = 90 * np.log(2.0)
    got = _np(_attn(sv, c))
    for i, n in enumerate(lens):
        # a score of 90 in units of 2: the scale in f32, the factor log2 e, their products: 6 roundings of 90, times log 2;
        # sums of n weights
        want = (n - 1) * 2.0 ** 10
        assert (np.abs(got[i] / want - 1) <= (6 * 90 + n + 40) * 2.0 ** -24).all(), (n, got[i].min(), got[i].max(), want)


def test_paged_attn_growing_maxima(sv):
    """Scores that rise over hundreds of units along the cache: the running maximum moves in every tile."""
    c = _attn_case(4, 2, 64, 16, [2000, 900], "f16", "rows")
    k = np.zeros((2000, 2, 64), np.float32)
    k[:, :, 0] = np.linspace(-60, 60, 2000)[:, None]
    k[:, :, 1] = _rng(1).standard_normal((2000, 2))
    for i, x in enumerate(c["lens"]):
        t = np.arange(x)
        for sign in (1,):
            c["kp"][_dev(c["table"][i][t // 16]).long(), _dev(t % 16)] = _dev(k[t] * sign).half()
    c["q"][:] = 0
    c["q"][:, :, 0] = [[5, -5, 1, 20], [2, 3, -20, 0]]
    c["q"][:, :, 1] = 1
    c["scale"] = 1.0
    _within(_attn(sv, c).cpu().numpy(), *_attn_ref(c))


def test_paged_attn_past_32_bits(sv):
    """Pages whose values lie past 2^32 bytes and 2^32 elements of the pool."""
    import torch

    ps, KV, hd, far = 16, 2, 128, 70000
    stride = 16 * ps * KV * hd  # pages of 128 KiB, a sixteenth of it used
    pool = torch.empty(2, far * stride, dtype=torch.float16, device="cuda")
    kp, vp = (x.as_strided((far, ps, KV, hd), (stride, KV * hd, hd, 1)) for x in pool)
    assert far * stride > 2 ** 32
    lens = [100, 30]
    small = _attn_case(8, KV, hd, ps, lens, "f16", "rows", spare=0)
    ids = _rng(2).permutation(np.arange(far - 1, far - 20, -1))[:small["kp"].shape[0]]
    kp[_dev(ids)], vp[_dev(ids)] = small["kp"], small["vp"]
    table = np.where(small["table"] >= 0, ids[small["table"]], -1).astype(np.int32)
    got = _attn(sv, {**small, "kp": kp, "vp": vp, "table": table})
    assert torch.equal(got, _attn(sv, small))
    r = _rng(8)
    k, v = (_dev(r.standard_normal((2, KV, hd)).astype(np.float32)) for _ in range(2))
    sv.paged_append_dev(k, v, kp, vp, _dev(table), _dev(np.array([99, 3], np.int32)))
    for i, p in enumerate((99, 3)):
        assert torch.equal(kp[int(table[i, p // ps]), p % ps], k[i].half())
        assert torch.equal(vp[int(table[i, p // ps]), p % ps], v[i].half())


# ---- log probabilities ------------------------------------------------------------


def _lp(sv, x, tokens, top, temperature):
    return sv.token_logprobs_dev(_dev(x), _dev(tokens), top=top, temperature=_opt(temperature))


def _lp_check(sv, x, tokens, top, temperature, what=""):
    lp, ent, ids, tops, b_lp, b_ent, b_top = ref.logprobs(x, tokens, top, temperature)
    got = [t.cpu().numpy() for t in _lp(sv, x, tokens, top, temperature)]
    assert (got[2] == ids).all(), (what, np.argwhere(got[2] != ids)[:5])
    for name, g, want, bound in (("lp", got[0], lp, b_lp), ("entropy", got[1], ent, b_ent), ("top", got[3], tops, b_top)):
        assert (np.isnan(g) == np.isnan(want)).all(), (what, name)
        want = np.where(want < -3.5e38, -np.inf, want)  # 2^128 and more: infinite in f32
        inf = np.isinf(want)
        assert (g[inf] == want[inf]).all(), (what, name)
        ok = np.isfinite(want)
        off = np.abs(g[ok].astype(np.float64) - want[ok]) - bound[ok]
        assert off.size == 0 or off.max() <= 0, (what, name, off.max())


LP = [(1, 1), (3, 2), (2, 63), (5, 255), (2, 1024), (3, 4096), (2, 4097), (4, 16384), (2, 16385), (7, 32000), (1, 32768),
      (1, 32769), (2, 151936), (150, 40001), (3, 300007), (520, 33000)]


@pytest.mark.parametrize("shape", LP, ids=lambda s: "x".join(map(str, s)))
def test_token_logprobs_match_their_definition(sv, shape):
    n, V = shape
    r = _rng(n, V)
    x = (r.standard_normal((n, V)) * 3).astype(np.float32)
    tokens = r.integers(0, V, n).astype(np.int32)
    t = (r.random(n) * 2 + 0.1).astype(np.float32)
    _lp_check(sv, x, tokens, 0, None)
    _lp_check(sv, x, tokens, 1, t)
    _lp_check(sv, x, tokens, 20, None)
    _lp_check(sv, x, tokens, 32, t)


@pytest.mark.parametrize("V", [100, 5000, 32000, 60000, 151936])
def test_token_logprobs_ties(sv, V):
    """Equal values, rows of them, both zeros, a few levels: the lower index first."""
    r = _rng(V)
    rows = [np.zeros(V), np.full(V, -3.5), r.integers(0, 3, V), r.integers(0, 40, V), np.where(r.random(V) < 0.5, 0.0, -0.0),
            np.arange(V) * 1e-3, -np.arange(V) * 1e-3, np.where(np.arange(V) == V - 1, 1.0, 0.0)]
    x = np.array(rows, np.float32)
    tokens = r.integers(0, V, len(x)).astype(np.int32)
    for top in (1, 7, 32):
        _lp_check(sv, x, tokens, top, None, top)


@pytest.mark.parametrize("V", [40, 5000, 32000, 151936])
def test_token_logprobs_masked_rows(sv, V):
    """-inf everywhere but for a few, but for none; NaN and infinities; padding tokens."""
    r = _rng(V, 1)
    x = np.full((9, V), -np.inf, np.float32)
    x[1, r.permutation(V)[:5]] = r.standard_normal(5)
    x[2, V - 1] = 4.0
    x[3] = r.standard_normal(V)
    x[3, r.permutation(V)[:V // 2]] = -np.inf
    x[4, :10] = np.nan
    x[5] = r.standard_normal(V)
    x[5, r.permutation(V)[:20]] = np.nan
    x[6] = np.nan
    x[7] = r.standard_normal(V)
    x[7, [3, 30]] = np.inf
    x[8] = -3.0e38
    x[8, 7] = 3.0e38
    for tokens in (r.integers(0, V, 9), np.full(9, 7), np.array([-1, V, 2 ** 31 - 1, -2 ** 31, 0, 1, 2, 3, 4])):
        for top in (0, 5, 32):
            _lp_check(sv, x, tokens.astype(np.int32), top, None, top)


@pytest.mark.parametrize("V", [700, 32000, 151936])
def test_token_logprobs_temperatures(sv, V):
    """Not positive, vanishing, infinite and NaN ones, with masked logits and with NaN."""
    r = _rng(V, 2)
    t = np.float32([1.0, 0.0, -1.0, 1e-39, np.inf, np.nan, 1e-3, 1e6, 0.5, 0.0, np.inf])
    x = r.standard_normal((len(t), V)).astype(np.float32)
    x[:, r.permutation(V)[:V // 3]] = -np.inf
    x[8, 5] = np.nan
    x[9, 5] = np.nan
    tokens = np.array([int(np.nanargmax(row)) if i % 2 else 11 for i, row in enumerate(x)], np.int32)
    for top in (0, 6):
        _lp_check(sv, x, tokens, top, t, top)


@pytest.mark.parametrize("V", [700, 20000, 32000, 40001, 151936])
def test_token_logprobs_of_logits_further_apart_than_f32_reaches(sv, V):
    """Finite logits whose difference passes f32's range, at temperatures at which it counts and at ordinary ones."""
    t = np.float32([np.inf, np.inf, 3.2e38, 1e38, 1e37, 2e36, 1e36, 1e31, 1e30, 9e29, 1.0, 0.5])
    x = (_rng(V, 4).uniform(-1, 1, (len(t), V)) * 3.4e38).astype(np.float32)
    x[1, :V - V // 3] = -3.4e38  # whole parts of a long row far below its maximum
    x[1, V - V // 3:] = 3.4e38
    x[2, :V // 2] = -3.3e38
    x[4, ::2] = -3.4e38
    x[4, 1::2] = 3.4e38
    tokens = np.array([0, V - 1] * (len(t) // 2), np.int32)
    for top in (0, 6):
        _lp_check(sv, x, tokens, top, t, top)
    x[:, 3::5] = -np.inf  # masked ones have no part in it
    for top in (0, 6):
        _lp_check(sv, x, tokens, top, t, top)


@pytest.mark.parametrize("V,threads", [(4000, 256), (32000, 256), (32000, 1024), (151936, 256)])
def test_token_logprobs_where_few_threads_hold_the_largest(sv, V, threads):
    """Every value of half of the threads above all others: more reach the bound than are collected."""
    r = _rng(V, 3)
    x = r.standard_normal((2, V)).astype(np.float32)
    own = (np.arange(V) // 4) % threads
    x[0, own % 64 < 32] += 50
    x[1, own % 64 < 32] = 7.0
    tokens = np.zeros(2, np.int32)
    for top in (3, 32):
        _lp_check(sv, x, tokens, top, None, top)


def test_token_logprobs_entropy_is_never_negative(sv):
    x = np.full((4, 40000), -40.0, np.float32)
    x[:, 5] = 30.0
    x[1, 6] = 29.9999
    x[2] = -100.0
    x[2, 9] = 0.0
    x[3] = -np.inf
    x[3, 0] = 1.0
    ent = _lp(sv, x, np.zeros(4, np.int32), 0, None)[1].cpu().numpy()
    assert (ent >= 0).all()
    _lp_check(sv, x, np.full(4, 5, np.int32), 3, None)


def test_token_logprobs_shapes_and_strides(sv):
    import torch

    import loom_amd

    r = _rng(6)
    x = _dev(r.standard_normal((2, 3, 500)).astype(np.float32))
    tok = _dev(r.integers(0, 500, (2, 3)).astype(np.int32))
    lp, ent, ids, tops = sv.token_logprobs_dev(x, tok, top=4)
    assert lp.shape == ent.shape == (2, 3) and ids.shape == tops.shape == (2, 3, 4)
    one = sv.token_logprobs_dev(x[1, 2], tok[1, 2], top=4)
    assert torch.equal(one[0], lp[1, 2]) and torch.equal(one[2], ids[1, 2])
    assert sv.token_logprobs_dev(x[:0], tok[:0], top=4)[2].shape == (0, 3, 4)
    # rows of a wider buffer, at odd places, through the C entry
    for V in (501, 33001):
        wide = _dev(r.standard_normal((5, V + 6)).astype(np.float32))
        flat = wide[:, 1:V + 1].contiguous()
        tok = _dev(r.integers(0, V, 5).astype(np.int32))
        want = sv.token_logprobs_dev(flat, tok, top=9)
        got = [torch.empty_like(t) for t in want]
        nb = loom_amd.lib().loomhip_token_logprobs_ws(5, V, 9)
        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device="cuda")
        loom_amd.check(loom_amd.lib().loomhip_token_logprobs_dev(
            wide.data_ptr() + 4, 5, V, V + 6, tok.data_ptr(), None, 9, *[t.data_ptr() for t in got], ws.data_ptr(), nb, None))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---- together ---------------------------------------------------------------------


class _Step:
    """One decode step of a batch over a paged cache: the projection's output in, log probabilities out."""

    def __init__(self, seed, n=5, H=8, KV=2, hd=64, ps=16, V=40000, kind="f16"):
        import torch

        r = _rng(seed)
        self.H, self.KV, self.hd, self.n = H, KV, hd, n
        self.lens = np.array([1, 17, 100, 333, 64][:n], np.int32)
        self.kp, self.vp = _cache(60, ps, KV, hd, kind, seed=seed)
        self.k0, self.v0, self.kind = self.kp.clone(), self.vp.clone(), kind
        self.table = _table(self.lens, ps, 60)
        self.qkv = _dev(r.standard_normal((n, (H + 2 * KV) * hd)).astype(np.float32))
        self.freqs = _dev(1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd))
        self.qn, self.kn = (_dev((1 + r.standard_normal(hd) * 0.1).astype(np.float32)) for _ in range(2))
        self.w = _dev(r.standard_normal((H * hd, V)).astype(np.float32) * 0.2)
        self.tok = _dev(r.integers(0, V, n).astype(np.int32))
        self.dtable, self.dlens = _dev(self.table), _dev(self.lens)
        self.dpos = _dev(self.lens - 1)
        torch.cuda.synchronize()

    def run(self, sv):
        import torch

        q, k, v = self.qkv.split((self.H * self.hd, self.KV * self.hd, self.KV * self.hd), 1)
        q = sv.paged_append_dev(k.unflatten(1, (self.KV, self.hd)), v.unflatten(1, (self.KV, self.hd)), self.kp, self.vp,
                                self.dtable, self.dpos, freqs=self.freqs, k_norm=self.kn, q=q.unflatten(1, (self.H, self.hd)),
                                q_norm=self.qn)
        o = sv.paged_attn_dev(q, self.kp, self.vp, self.dtable, self.dlens, self.hd ** -0.5)
        logits = torch.matmul(o.flatten(1), self.w)
        return (q, o, logits) + sv.token_logprobs_dev(logits, self.tok, top=5)


def test_a_decode_step_over_a_paged_cache(sv):
    s = _Step(1)
    q, o, logits, lp, ent, ids, tops = s.run(sv)
    x = _np(s.qkv)
    H, KV, hd = s.H, s.KV, s.hd
    want, bound = ref.norm_rope(x[:, :H * hd].reshape(-1, H, hd), s.lens - 1, _np(s.freqs), _np(s.qn), 1e-6, False)
    _within(_np(q), want, bound, "q")
    k, kb = ref.norm_rope(x[:, H * hd:(H + KV) * hd].reshape(-1, KV, hd), s.lens - 1, _np(s.freqs), _np(s.kn), 1e-6, False)
    for i, at in enumerate(ref.slots(s.table, 60, 16, s.lens - 1, None)):
        _within(_np(s.kp[at]), k[i], ref.rounded(k[i], kb[i], s.kind), "k")
        s.k0[at], s.v0[at] = s.kp[at], s.qkv[i, (H + KV) * hd:].view(KV, hd).half()
    assert (s.kp == s.k0).all() and (s.vp == s.v0).all()
    _within(_np(o), *ref.attn(_np(q), _np(s.kp), _np(s.vp), s.table, s.lens, hd ** -0.5, 0), "o")
    wl, we, wi, wt, bl, be, bt = ref.logprobs(_np(logits), s.tok.cpu().numpy(), 5, None)
    assert (ids.cpu().numpy() == wi).all()
    _within(_np(lp), wl, bl), _within(_np(ent), we, be), _within(_np(tops), wt, bt)


def test_prefill_then_shared_prefix_attention_agrees(sv):
    """Rotated queries and keys serve prefix_attn_dev's contiguous rows as they serve the pages."""
    r = _rng(12)
    n, H, KV, hd, ps, T = 3, 8, 2, 64, 16, 50
    k, v = (_dev(r.standard_normal((n * T, KV, hd)).astype(np.float32)) for _ in range(2))
    q = _dev(r.standard_normal((n * T, H, hd)).astype(np.float32))
    pos = _dev(np.tile(np.arange(T), n).astype(np.int32))
    lanes = _dev(np.repeat(np.arange(n), T).astype(np.int32))
    freqs = _dev(1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd))
    kp, vp = _cache(12, ps, KV, hd, "f16")
    table = _table([T] * n, ps, 12)
    q1 = sv.paged_append_dev(k, v, kp, vp, _dev(table), pos, lanes=lanes, freqs=freqs, q=q)
    q2, k2 = sv.qk_norm_rope_dev(q, k, pos, freqs)
    assert (q1 == q2).all()
    last = q2.view(n, T, H, hd)[:, -1].contiguous()
    lens = _dev(np.full(n, T, np.int32))
    a = sv.paged_attn_dev(last, kp, vp, _dev(table), lens, hd ** -0.5)
    kh, vh = k2.half().view(n, T, KV, hd), v.half().view(n, T, KV, hd)
    b = sv.prefix_attn_dev(last.unsqueeze(1), None, None, kh, vh, lens, hd ** -0.5)[:, 0]
    want, bound = ref.attn(_np(last), _np(kp), _np(vp), table, [T] * n, hd ** -0.5, 0)
    _within(_np(a), want, bound), _within(_np(b), want, bound)


def test_the_step_captured_and_replayed(sv):
    """Every replay reads the inputs that are there then, with eager work and synchronizations in between."""
    import torch

    s = _Step(2)
    s.run(sv)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = s.run(sv)
    for seed in range(4):
        other = _Step(20 + seed)
        s.qkv.copy_(other.qkv)
        s.dlens.copy_(_dev(np.maximum(s.lens - 3 * seed, 1).astype(np.int32)))
        s.dpos.copy_(s.dlens - 1)
        s.kp.copy_(other.kp), s.vp.copy_(other.vp)
        s.dtable.copy_(_dev(_table(s.lens, 16, 60, seed=seed)))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out] + [s.kp.clone(), s.vp.clone()]
        s.kp.copy_(other.kp), s.vp.copy_(other.vp)
        want = list(s.run(sv)) + [s.kp, s.vp]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_steps_on_two_streams_and_threads(sv):
    import threading

    import torch

    steps = [_Step(31), _Step(32)]
    want = [[t.clone() for t in s.run(sv)] for s in steps]
    torch.cuda.synchronize()
    out = [None, None]

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                out[i] = steps[i].run(sv)
        st.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(out, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_paged_refusals_raise(sv):
    import torch

    import loom_amd

    c = _attn_case(8, 2, 64, 16, [30, 40], "f16", "rows")
    with pytest.raises(loom_amd.LoomHipError, match="declined|not served"):
        q = torch.zeros(2, 8, 60, device="cuda")
        kp = torch.zeros(5, 16, 2, 60, device="cuda", dtype=torch.float16)
        sv.paged_attn_dev(q, kp, kp, _dev(c["table"]), _dev(c["lens"]), 1.0)
    with pytest.raises(loom_amd.LoomHipError, match="table of"):
        sv.paged_attn_dev(_dev(c["q"]), c["kp"], c["vp"], _dev(c["table"][:1]), _dev(c["lens"]), 1.0)
    with pytest.raises(ValueError, match="tensors on"):
        sv.paged_attn_dev(_dev(c["q"]), c["kp"], c["vp"], torch.from_numpy(c["table"]), _dev(c["lens"]), 1.0)
    with pytest.raises(loom_amd.LoomHipError, match="not served"):
        sv.token_logprobs_dev(torch.zeros(1, 100, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32), top=33)
    x = torch.zeros(4, 8, 64, device="cuda")
    with pytest.raises(loom_amd.LoomHipError, match="overlaps"):
        sv.qk_norm_rope_dev(x[:, :4], x[:, 4:], torch.zeros(4, device="cuda", dtype=torch.int32), None, q_out=x[:, 2:6])
