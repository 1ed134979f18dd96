"""Every form of the batched serving kernels on the device: over ranges of many
tiles, where the running maximum moves in mid-range, and to f32's precision
(serving_forms.py)."""
import numpy as np
import pytest

import serving_forms as sf
from test_gpu_serving import _attn_case, _dev, _within, sv  # noqa: F401

pytestmark = pytest.mark.gpu

ATTN_SHAPES = [s for s, _ in sf.ATTN_FORMS.values()] + sf.ATTN_MORE
ids = lambda s: "x".join(map(str, s))  # noqa: E731


def _run(sv, c, ragged):
    args = [_dev(c[k]) for k in ("q", "kp", "vp", "ko", "vo", "own_len")]
    return sv.prefix_attn_dev(*args, c["scale"], q_len=_dev(c["q_len"]) if ragged else None)


@pytest.mark.parametrize("shape", ATTN_SHAPES + [sf.ATTN_LONG], ids=ids)
def test_attention_forms_hold_f32s_precision(sv, shape):
    c = sf.attn_case(shape)
    for ragged in (True, False):
        want, bound = sf.attn(c, ragged)
        got = _run(sv, c, ragged).cpu().numpy()
        _within(got, want, bound, f"ragged {ragged}")
        assert (got[np.isnan(want)] == 0).all()


def _check_dense(sv, c, ragged):
    """Against the definition in 64 bits on the device, within the bound of serving_ref.prefix_attn."""
    import torch

    q, kp, vp, ko, vo = (torch.from_numpy(np.asarray(c[k], np.float64)).cuda() for k in ("q", "kp", "vp", "ko", "vo"))
    n, nq, heads, hd = q.shape
    kv = kp.shape[1]
    G, P = heads // kv, len(kp)
    got = _run(sv, c, ragged).double()
    for i in range(n):
        L = int(c["q_len"][i]) if ragged else nq
        length = int(c["own_len"][i])
        seen = torch.arange(L, device="cuda") + length - L + 1
        hidden = torch.arange(length, device="cuda")[None, :] >= seen[:, None]  # [L][length]
        assert bool((got[i, L:] == 0).all())
        for h in range(kv if L else 0):
            k, v = torch.cat([kp[:, h], ko[i, :length, h]]), torch.cat([vp[:, h], vo[i, :length, h]])
            qi = q[i, :L, h * G:(h + 1) * G].reshape(L * G, hd)
            s, size = qi @ k.t().contiguous() * c["scale"], qi.abs() @ k.abs().t().contiguous() * abs(c["scale"])
            s, size = s.view(L, G, -1), size.view(L, G, -1)
            s[:, :, P:].masked_fill_(hidden[:, None, :], -np.inf)
            size[:, :, P:].masked_fill_(hidden[:, None, :], 0.0)
            T = P + seen.clamp(min=0).double()
            p = torch.softmax(s, -1).view(L * G, -1)
            want, mag = (p @ v).view(L, G, hd), (p @ v.abs()).view(L, G, hd)
            b = 2 * (hd + 8) * size.amax(-1) + 36 + 2 * T[:, None]
            off = (got[i, :L, h * G:(h + 1) * G] - want).abs() - sf.EPS * b[:, :, None] * mag
            assert float(off.max()) <= 0, (i, h, float(off.max()))


@pytest.mark.parametrize("shape", ATTN_SHAPES, ids=ids)
def test_attention_forms_match_the_definition(sv, shape):
    c = _attn_case(*shape)
    for ragged in (True, False):
        _check_dense(sv, c, ragged)


@pytest.mark.parametrize("shape", ATTN_SHAPES, ids=ids)
def test_attention_forms_where_the_maximum_moves(sv, shape):
    """Scores that step up by 10 (e^10 > 2^14, the room that weights have) every 100 rows, in mid-tile and mid-range, and
    the other way around for every second query head."""
    c = _attn_case(*shape)
    heads, P, n, own = shape[0], shape[3], shape[4], shape[6]
    q = c["q"] * np.float32(np.sqrt(shape[2]))
    q[..., 0] = np.where(np.arange(heads) % 2, -1.0, 1.0) * np.sqrt(shape[2])
    c["q"] = (q / np.float32(3)).astype(np.float32)  # scores of the other elements within a few units
    c["kp"][..., 0] = (np.arange(P) // 100 * 30)[:, None]
    c["ko"][..., 0] = ((P + np.arange(own)) // 100 * 30)[None, :, None]
    for ragged in (True, False):
        _check_dense(sv, c, ragged)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", sf.LORA_FORMS, ids=ids)
def test_adapter_forms_hold_f32s_precision(sv, shape, dtype):
    import torch

    c = sf.lora_case(shape)
    want, bound = sf.lora(c)
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]  # all hold a and b exactly
    for order in (np.arange(shape[0]), np.argsort(c["ids"], kind="stable")):  # mixed, and each adapter's together
        got = sv.lora_dev(_dev(c["x"][order]), _dev(c["a"], t), _dev(c["b"], t), _dev(c["scale"]), _dev(c["ids"][order]),
                          base=_dev(c["base"][order]))
        _within(got.cpu().numpy(), want[order], bound[order], dtype)
