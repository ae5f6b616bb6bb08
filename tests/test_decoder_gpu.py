"""The decoder whose continuations share a prompt (cached rows, windowed and
full layers, scoring, gradient, generation) against each sequence computed
whole from scratch in f64 with dense masks and the chain's rounding points."""

import numpy as np
import pytest
import torch

from forma_b200 import api
from forma_b200.decoder import Decoder, DecoderConfig
from oracle.vit import f32, gelu_tanh, low

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(vocab=500, embed=256, heads=4, kv_heads=2, layers=3, mlp=512, window=16, sinks=2, positions=256)


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def whole(dec: Decoder, tokens: np.ndarray):
    """Normed hidden rows and logits of whole sequences, int [G, N]."""
    cfg = dec.cfg
    G, N = tokens.shape
    H, K, D, E = cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.embed
    at = np.arange(N)
    seen = at[None, :] <= at[:, None]
    near = seen & ((at[None, :] > at[:, None] - cfg.window) | (at[None, :] < cfg.sinks))

    def norm(t):
        m = t.mean(-1, keepdims=True)
        return low(f32((t - m) / np.sqrt(t.var(-1, keepdims=True) + cfg.eps)))

    def weight(w):
        return f64(w)[:, :, 0, 0].T

    x = f32(f64(dec.embedding)[tokens] + f64(dec.position)[:N])
    for i, blk in enumerate(dec.blocks):
        qkv = low(norm(x) @ weight(blk["qkv"])).reshape(G, N, H + 2 * K, D).transpose(0, 2, 1, 3)
        q, k, v = qkv[:, :H], np.repeat(qkv[:, H:H + K], H // K, 1), np.repeat(qkv[:, H + K:], H // K, 1)
        s = np.where(seen if cfg.full(i) else near, q @ k.transpose(0, 1, 3, 2) / np.sqrt(D), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        a = low((p / p.sum(-1, keepdims=True)) @ v).transpose(0, 2, 1, 3).reshape(G, N, E)
        x = f32(x + a @ weight(blk["proj"]))
        x = f32(x + low(gelu_tanh(f32(norm(x) @ weight(blk["fc1"])))) @ weight(blk["fc2"]))
    h = norm(x)
    return h, low(h @ weight(dec.head))


def setup(cuda, P, G, L, seed):
    g = torch.Generator().manual_seed(seed)
    dec = Decoder(CFG, cuda, seed=seed)
    prompt = torch.randint(CFG.vocab, (P,), generator=g, dtype=torch.int32)
    own = torch.randint(CFG.vocab, (G, L), generator=g, dtype=torch.int32)
    both = np.concatenate([np.broadcast_to(prompt.numpy(), (G, P)), own.numpy()], axis=1)
    return dec, prompt.to(cuda), own.to(cuda), both


@pytest.mark.parametrize("P,G,L", [(1, 3, 5), (11, 2, 40), (90, 5, 33), (150, 1, 1)])
def test_scores_match_whole_sequences(cuda, P, G, L):
    dec, prompt, own, both = setup(cuda, P, G, L, P)
    targets = torch.roll(own, -1, 1)
    targets[:, -1] = api.NO_TOKEN
    state = dec.start(dec.read(prompt), G, L)
    scored, logits, hidden = dec.score(state, own, targets, top=7)
    assert api.device_status() == 0
    ref = whole(dec, both)[1][:, P:]
    got = f64(logits)
    err = np.abs(got - ref).max()
    assert err <= 2e-2 * np.abs(ref).max(), err  # bf16 tensor-core gate, applied to the chain's output
    # probabilities of the logits that were scored
    m = got.max(-1, keepdims=True)
    lp = got - m - np.log(np.exp(got - m).sum(-1, keepdims=True))
    t = targets.cpu().numpy()
    exp = np.where(t < 0, 0.0, np.take_along_axis(lp, np.maximum(t, 0)[..., None], -1)[..., 0])
    # lse of ~10 in f32 (2^-23 * 16) and approximate base-2 exponentials (2^-22): below 1e-5
    assert np.abs(f64(scored.logprob) - exp).max() <= 1e-5
    assert np.abs(f64(scored.entropy) + (np.exp(lp) * lp).sum(-1)).max() <= 1e-4
    order = np.argsort(-got, axis=-1, kind="stable")[..., :7]
    assert np.array_equal(scored.top_index.cpu().numpy(), order)


@pytest.mark.parametrize("P,G,steps", [(5, 2, 30), (90, 3, 9)])
def test_generation_is_the_likeliest_continuation(cuda, P, G, steps):
    """Each generated token is, by the whole-sequence reference, within the
    chain's gate of the likeliest one; and scoring what was generated in one
    call gives the log probabilities of the single steps."""
    dec, prompt, own, _ = setup(cuda, P, G, 1, 7 + P)
    read = dec.read(prompt)
    tokens, scores = dec.generate(dec.start(read, G, steps), own[:, 0], steps)
    assert api.device_status() == 0
    inputs = torch.cat([own, tokens[:, :-1]], 1)
    both = np.concatenate([np.broadcast_to(prompt.cpu().numpy(), (G, P)), inputs.cpu().numpy()], axis=1)
    ref = whole(dec, both)[1][:, P:]
    gate = 2e-2 * np.abs(ref).max()
    picked = np.take_along_axis(ref, tokens.cpu().numpy()[..., None], -1)[..., 0]
    assert (picked >= ref.max(-1) - 2 * gate).all()
    again, _, _ = dec.score(dec.start(read, G, steps), inputs, tokens)
    # a log probability moves by at most twice the largest change of a logit
    assert np.abs(f64(again.logprob) - f64(scores)).max() <= 4 * gate


def test_ragged_continuations_extend_from_their_own_ends(cuda):
    """Caches of different lengths: after one padded call the lengths are set
    back to the real ones, and the next token lands behind each own end."""
    P, G, L = 60, 3, 12
    dec, prompt, own, _ = setup(cuda, P, G, L, 21)
    real = torch.tensor([12, 1, 5], dtype=torch.int32, device=cuda)
    state = dec.start(dec.read(prompt), G, L + 1)
    dec.extend(state, own)
    state.lengths = real.clone()
    nxt = torch.tensor([[3], [4], [5]], dtype=torch.int32, device=cuda)
    got = f64(dec.logits(dec.extend(state, nxt)))[:, 0]
    for s, n in enumerate(real.tolist()):
        row = np.concatenate([prompt.cpu().numpy(), own[s, :n].cpu().numpy(), nxt[s].cpu().numpy()])
        ref = whole(dec, row[None])[1][0, -1]
        assert np.abs(got[s] - ref).max() <= 2e-2 * np.abs(ref).max()


def test_head_gradient(cuda):
    P, G, L = 20, 4, 9
    dec, prompt, own, _ = setup(cuda, P, G, L, 33)
    targets = torch.roll(own, -1, 1)
    targets[:, -1] = api.NO_TOKEN
    gl = torch.randn(G, L, generator=torch.Generator().manual_seed(1)).to(cuda)
    ge = torch.full((G, L), 0.25, device=cuda)
    scored, logits, hidden = dec.score(dec.start(dec.read(prompt), G, L), own, targets)
    x, h = f64(logits).reshape(G * L, -1), f64(hidden).reshape(G * L, -1)
    grad = f64(dec.head_gradient(scored, logits, hidden, targets, gl, ge))
    assert api.device_status() == 0
    m = x.max(-1, keepdims=True)
    lp = x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))
    p = np.exp(lp)
    t = targets.cpu().numpy().reshape(-1)
    hot = (np.arange(x.shape[1])[None] == t[:, None])
    g1 = np.where(t < 0, 0.0, f64(gl).reshape(-1))[:, None]
    d = g1 * (hot - p) - 0.25 * p * (lp - (p * lp).sum(-1, keepdims=True))
    ref = d.T @ h
    # each element of the logits' gradient is rounded to bf16 (2^-9 of itself, plus f32 work); sums in f32
    bound = 2.0 ** -8 * (np.abs(d).T @ np.abs(h)) + 1e-6
    assert (np.abs(grad - ref) <= bound).all()


def test_routes(cuda):
    """The example's calls take the tensor-core and streaming kernels."""
    dec, prompt, own, _ = setup(cuda, 90, 5, 33, 3)
    state = dec.start(dec.read(prompt), 5, 33)
    q = torch.zeros(5, 4, 33, 64, dtype=torch.bfloat16, device=cuda)
    pk, pv = state.prompt.layers[1]
    ck, cv = state.caches[1]
    api.attention_prefix(q, pk, pv, ck, cv)
    assert any(r.startswith("span_tile_kernel<64") for r in api.last_route()), api.last_route()
    api.token_logprobs(torch.zeros(4, 500, dtype=torch.bfloat16, device=cuda))
    assert any("token_stream_kernel" in r for r in api.last_route()), api.last_route()
