"""The batched serving operators beside the frame: a Decoder's caches and logits
as they lie, and one speculative step in the order the documentation gives."""
import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving import _dev, _rng, _within, sv  # noqa: F401

pytestmark = pytest.mark.gpu

P, K = 40, 3  # rows of the shared prefix, drafted tokens


@pytest.fixture(scope="module")
def decoded(sv):
    """Four lanes of a small Qwen3-shaped model after K + 1 steps over a context of 60 rows, in caches of 128: the
    decoder, and the logits and greedy tokens of every step."""
    from loom_amd import frame

    spec = frame.qwen3_30b_a3b(ctx_len=128, n_layers=2, vocab=4096, n_expert=16)
    dec = frame.Decoder(frame.DeviceModel.synth(spec, seed=5), 4)
    dec.prefill_random(60, seed=3)
    dec.tokens.copy_(_dev(np.array([1, 77, 900, 4000], np.int32)))
    logits, tokens = [], []
    for _ in range(K + 1):
        dec.step()
        logits.append(dec.logits.clone())
        tokens.append(dec.tokens.clone())
    return dec, logits, tokens


def _caches(dec, layer, rows):
    """Lane 0's first P rows as the prefix, the other lanes' caches cut to `rows`."""
    s = dec.model.spec
    k, v = (c[:, layer].unflatten(-1, (s.n_kv_heads, s.head_dim)) for c in (dec.k_cache, dec.v_cache))
    return k[0, :P], v[0, :P], k[1:, :rows], v[1:, :rows]


@pytest.mark.parametrize("layer", [0, 1])
def test_a_decoders_caches(sv, decoded, layer):
    """Whole lanes of ctx_len rows, and cut to the longest length: the rows behind are the same to the result."""
    dec, _, _ = decoded
    assert dec.pos.tolist() == [60 + K + 1] * 4
    own_len = (dec.pos[1:] - _dev(np.array([0, 20, 63], np.int32))).contiguous()
    q = _rng(layer, 9).standard_normal((3, 2, 32, 128)).astype(np.float32)
    host = [t.contiguous().cpu().numpy().view(np.float16) for t in _caches(dec, layer, 128)]
    want, bound = ref.prefix_attn(q, *host, own_len.cpu().numpy(), None, 128 ** -0.5)
    for rows in (128, int(own_len.max())):
        got = sv.prefix_attn_dev(_dev(q), *_caches(dec, layer, rows), own_len, 128 ** -0.5)
        _within(got.cpu().numpy(), want, bound, f"{rows} rows")


def test_the_frames_greedy_pick(sv, decoded):
    """Probabilities of a decoder's logits at a temperature of zero: one at the token that the frame picked."""
    import torch

    dec, logits, tokens = decoded
    for lg, tok in zip(logits, tokens):
        p = sv.token_probs_dev(lg, torch.zeros(4, device="cuda"))
        assert bool((p.argmax(-1).to(torch.int32) == tok).all()) and bool((p.sum(-1) == 1).all())
        want, bound = ref.token_probs(lg.cpu().numpy(), None)
        _within(sv.token_probs_dev(lg).cpu().numpy(), want, bound)


def test_one_speculative_step(sv, decoded):
    """Projection, adapters over its output, attention, probabilities, verification; the drafts are the frame's own
    greedy tokens, so at a temperature of zero all are accepted and the next is its next."""
    import torch

    from loom_amd import Q4_K
    from loom_amd.backend import matvec_dev, repack_dev, synth_ggml_dev

    dec, step_logits, tokens = decoded
    n, k, heads, hd, rows, cols, vocab = 3, K, 32, 128, 4096, 2048, 4096
    r = torch.Generator(device="cuda").manual_seed(4)
    w = repack_dev(Q4_K, synth_ggml_dev(Q4_K, rows, cols, 1, 3, 0.02), rows, cols, 1)
    x = torch.randn(n * (k + 1), cols, generator=r, device="cuda")
    a = (torch.randn(4, 16, cols, generator=r, device="cuda") / cols ** 0.5).half()
    b = (torch.randn(4, rows, 16, generator=r, device="cuda") / 4).half()
    scale = torch.ones(4, device="cuda")
    ids = torch.arange(-1, n * (k + 1) - 1, device="cuda", dtype=torch.int32) % 5
    k_prefix, v_prefix, k_own, v_own = _caches(dec, 1, 128)
    own_len, q_len = dec.pos[1:].contiguous(), torch.full((n,), k + 1, dtype=torch.int32, device="cuda")
    logits = torch.stack(step_logits, 1)[1:].reshape(n * (k + 1), vocab)
    drafts = torch.stack(tokens[:k], 1)[1:].contiguous()
    u_accept, u_sample = torch.rand(n, k, generator=r, device="cuda"), torch.rand(n, generator=r, device="cuda")

    q = torch.empty(n * (k + 1), rows, device="cuda")
    matvec_dev(Q4_K, q, w, x, n * (k + 1), rows, cols)
    plain = q.clone()
    sv.lora_dev(x, a, b, scale, ids, base=q, out=q)
    o = sv.prefix_attn_dev(q.view(n, k + 1, heads, hd), k_prefix, v_prefix, k_own, v_own, own_len, hd ** -0.5, q_len=q_len)
    p = sv.token_probs_dev(logits, torch.zeros(n * (k + 1), device="cuda"))
    got, accepted = sv.verify_drafts_dev(p.view(n, k + 1, vocab), drafts, u_accept, u_sample)

    want, bound = ref.lora(*(t.float().cpu().numpy() for t in (x, a, b, scale)), ids.cpu().numpy(), plain.cpu().numpy())
    _within(q.cpu().numpy(), want, bound, "adapters")
    host = [t.contiguous().cpu().numpy().view(np.float16) for t in (k_prefix, v_prefix, k_own, v_own)]
    want, bound = ref.prefix_attn(q.view(n, k + 1, heads, hd).cpu().numpy(), *host, own_len.cpu().numpy(), None, hd ** -0.5)
    _within(o.cpu().numpy(), want, bound, "attention")
    assert accepted.tolist() == [k] * n
    assert bool((got == torch.stack(tokens, 1)[1:]).all())
