"""A decoder whose continuations share one prompt, chained from the operator API.

The language-model workload of the span-attention and token-probability
operators: a prompt is read once, many continuations of it are scored (log
probability and entropy of every token, the likeliest alternatives), trained
on, or extended a token at a time.  Pre-norm blocks, every `full_every`-th
with attention over everything and the others with a window::

    x  = embedding[token] + position
    for each layer:
        h  = LN(x)                           layer_norm, rounded to the low dtype as stored
        q, k, v = heads(h W_qkv)             GEMM rounded in its epilogue; few key/value heads
        k, v -> the sequence's cache rows
        x  = x + concat_heads(a) W_o         a = attention_window(q, cache) or
                                             attention_prefix(q, prompt's keys, cache)
        h  = LN(x);  x = x + GELU(h W_1) W_2
    logits = LN(x) W_head                    low dtype; token_logprobs, token_logprobs_grad

Caches.  A full layer's prompt keys are stored once, whatever the number of
continuations, and shared by their rows in every call (attention_prefix).  A windowed layer
sees only its first `sinks` and last `window` positions, so each continuation
starts from a copy of the prompt's first `sinks` and last `window - 1` rows:
dropping the rows between shifts the positions of what follows by one amount
and leaves every visible (query, key) pair in place.

Tokens live as channels-last rows, so every projection is a 1x1 convolution
that reads them in place.  Weights are random (seeded); no checkpoint is
involved.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from . import api
from .api import ConvOptions, TokenLogprobs

_ONE = ConvOptions([1, 1], [1, 1], [0, 0], [0, 0])  # 1x1, stride 1, no padding


@dataclass(frozen=True)
class DecoderConfig:
    vocab: int = 32000
    embed: int = 1024
    heads: int = 16
    kv_heads: int = 4
    layers: int = 4
    mlp: int = 4096
    full_every: int = 2   # layers 1, 3, .. see everything; the others a window
    window: int = 256
    sinks: int = 4
    positions: int = 8192
    eps: float = 1e-5

    @property
    def head_dim(self) -> int:
        return self.embed // self.heads

    def full(self, layer: int) -> bool:
        return layer % self.full_every == self.full_every - 1


@dataclass
class Prompt:
    """The prompt's rows of each layer's cache: [Hkv, P, D] in full layers,
    the rows that a window can still reach in the others."""

    length: int
    layers: List[Tuple[torch.Tensor, torch.Tensor]]


@dataclass
class Continuations:
    """Caches of `sequences` continuations of one prompt.  ``lengths`` (int32
    [G]) counts each one's own tokens; it may be set back, or replaced."""

    prompt: Prompt
    caches: List[Tuple[torch.Tensor, torch.Tensor]]  # [G, Hkv, rows, D]
    kept: List[int]                                  # prompt rows at the front of each cache
    lengths: torch.Tensor
    _known: Optional[tuple] = None                   # lengths that the host knows: (tensor, its version, their maximum)

    @property
    def room(self) -> int:
        """Own tokens that every layer's cache holds."""
        return min(c[0].shape[2] - n for c, n in zip(self.caches, self.kept))

    def require(self, sequences: int, tokens: int, positions: int) -> int:
        """The longest continuation's tokens, if ``tokens`` more fit each one's
        cache and the model's ``positions``; ValueError otherwise.  Past the
        room a cache would be indexed out of range on the device, which ends the
        process's context.  The device is read only where `lengths` were set
        from outside."""
        G = self.lengths.shape[0]
        if sequences != G:
            raise ValueError(f"tokens of {sequences} continuations for caches of {G}")
        if self._known is None or self._known[0] is not self.lengths or self._known[1] != self.lengths._version:
            low, high = (int(x) for x in self.lengths.aminmax()) if G else (0, 0)
            if low < 0 or high > self.room:
                raise ValueError(f"lengths {low} to {high} for caches of {self.room} tokens")
            self._known = (self.lengths, self.lengths._version, high)
        longest = self._known[2]
        if longest + tokens > self.room:
            raise ValueError(f"{tokens} tokens behind {longest} exceed the caches' room of {self.room}")
        if self.prompt.length + longest + tokens > positions:
            raise ValueError(f"position {self.prompt.length + longest + tokens - 1} exceeds the model's {positions}")
        return longest

    def advance(self, tokens: int, longest: int) -> None:
        self.lengths = self.lengths + tokens
        self._known = (self.lengths, self.lengths._version, longest + tokens)


class Decoder:
    def __init__(self, cfg: DecoderConfig, device, dtype=torch.bfloat16, seed: int = 0):
        self.cfg, self.dtype, self.device = cfg, dtype, torch.device(device)
        g = torch.Generator(device="cpu").manual_seed(seed)
        E, M, D = cfg.embed, cfg.mlp, cfg.head_dim

        def w(o, i):
            return (torch.randn(o, i, 1, 1, generator=g) / math.sqrt(i)).to(dtype).to(self.device)

        self.embedding = torch.randn(cfg.vocab, E, generator=g).to(self.device)
        self.position = (torch.randn(cfg.positions, E, generator=g) * 0.02).to(self.device)
        self.blocks = [{"qkv": w((cfg.heads + 2 * cfg.kv_heads) * D, E), "proj": w(E, E), "fc1": w(M, E), "fc2": w(E, M)}
                       for _ in range(cfg.layers)]
        self.head = w(cfg.vocab, E)

    # -- pieces

    @staticmethod
    def _rows(x: torch.Tensor) -> torch.Tensor:
        """Rows [.., C] as the logical [1, C, 1, rows] input (or output) of a 1x1 convolution."""
        return x.view(1, 1, -1, x.shape[-1]).permute(0, 3, 1, 2)

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        return api.layer_norm_low(x, [x.dim() - 1], self.cfg.eps, self.dtype)

    def _project(self, h: torch.Tensor, weight: torch.Tensor, fn=api.conv_low_into) -> torch.Tensor:
        out = torch.empty(*h.shape[:-1], weight.shape[0], dtype=self.dtype, device=h.device)
        fn(self._rows(h), weight, _ONE, self._rows(out))
        return out

    def _embed(self, tokens: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        return api.add(self.embedding[tokens.long()], self.position[positions.long()])

    def _run(self, x: torch.Tensor, attend) -> torch.Tensor:
        """The blocks over x [G, L, E] (f32, added into).  ``attend(layer, q,
        k, v, out)`` gets head views of the fused projection and writes [G, H,
        L, D]."""
        cfg = self.cfg
        G, L, E = x.shape
        H, K, D = cfg.heads, cfg.kv_heads, cfg.head_dim
        for i, blk in enumerate(self.blocks):
            qkv = self._project(self._norm(x), blk["qkv"]).view(G, L, H + 2 * K, D).transpose(1, 2)
            a = torch.empty(G, L, E, dtype=self.dtype, device=x.device)
            attend(i, qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], a.view(G, L, H, D).transpose(1, 2))
            api.conv_low_f32_accumulate(self._rows(a), blk["proj"], _ONE, self._rows(x))
            m = self._project(self._norm(x), blk["fc1"], api.conv_low_gelu_into)
            api.conv_low_f32_accumulate(self._rows(m), blk["fc2"], _ONE, self._rows(x))
        return x

    # -- the workload

    def read(self, tokens: torch.Tensor) -> Prompt:
        """Reads one prompt (int32 [P]) and keeps what its continuations need of it."""
        cfg, P = self.cfg, tokens.shape[0]
        if P > cfg.positions:
            raise ValueError(f"a prompt of {P} tokens exceeds the model's {cfg.positions} positions")
        kept: List[Tuple[torch.Tensor, torch.Tensor]] = []

        def attend(layer, q, k, v, out):
            # with a window as long as the prompt every earlier key is visible
            api.attention_window(q, k, v, max(P, 1) if cfg.full(layer) else cfg.window,
                                 0 if cfg.full(layer) else cfg.sinks, out=out)
            if cfg.full(layer) or P <= cfg.sinks + cfg.window - 1:
                kept.append((k[0].contiguous(), v[0].contiguous()))
            else:
                tail = P - (cfg.window - 1)
                kept.append(tuple(torch.cat([t[0, :, :cfg.sinks], t[0, :, tail:]], dim=1) for t in (k, v)))

        self._run(self._embed(tokens, torch.arange(P, device=self.device))[None], attend)
        return Prompt(P, kept)

    def start(self, prompt: Prompt, sequences: int, room: int) -> Continuations:
        """Empty caches for ``sequences`` continuations of up to ``room`` tokens each."""
        caches, kept = [], []
        for layer, rows in enumerate(prompt.layers):
            n = 0 if self.cfg.full(layer) else rows[0].shape[1]
            pair = []
            for t in rows:
                c = torch.empty(sequences, t.shape[0], n + room, t.shape[2], dtype=t.dtype, device=t.device)
                c[:, :, :n] = t[:, :n]
                pair.append(c)
            caches.append(tuple(pair))
            kept.append(n)
        return Continuations(prompt, caches, kept, torch.zeros(sequences, dtype=torch.int32, device=self.device))

    def extend(self, state: Continuations, tokens: torch.Tensor) -> torch.Tensor:
        """Appends tokens (int32 [G, L]) to every continuation and returns their
        normed hidden rows [G, L, E] in the low dtype.  ValueError, with nothing
        changed, where they do not fit."""
        cfg = self.cfg
        G, L = tokens.shape
        longest = state.require(G, L, cfg.positions)
        at = state.lengths[:, None].long() + torch.arange(L, device=self.device)  # place among the own tokens
        state.advance(L, longest)
        seq = torch.arange(G, device=self.device)[:, None]

        def attend(layer, q, k, v, out):
            ck, cv = state.caches[layer]
            n = state.kept[layer]
            ck[seq, :, at + n] = k.transpose(1, 2)
            cv[seq, :, at + n] = v.transpose(1, 2)
            if cfg.full(layer):
                pk, pv = state.prompt.layers[layer]
                api.attention_prefix(q, pk, pv, ck, cv, state.lengths, out=out)
            else:
                api.attention_window(q, ck, cv, cfg.window, cfg.sinks, state.lengths + n, out=out)

        x = self._run(self._embed(tokens, at + state.prompt.length), attend)
        return self._norm(x)

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return self._project(hidden, self.head)

    def score(self, state: Continuations, tokens: torch.Tensor, targets: torch.Tensor,
              top: int = 0) -> Tuple[TokenLogprobs, torch.Tensor, torch.Tensor]:
        """Appends ``tokens`` and scores ``targets`` (both int32 [G, L];
        NO_TOKEN where a shorter continuation has ended): the probabilities,
        the logits and the hidden rows they came from."""
        hidden = self.extend(state, tokens)
        logits = self.logits(hidden)
        return api.token_logprobs(logits, targets, top), logits, hidden

    def head_gradient(self, scored: TokenLogprobs, logits: torch.Tensor, hidden: torch.Tensor, targets: torch.Tensor,
                      grad_logprob: torch.Tensor, grad_entropy: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Gradient [V, E] (f32) for the head's weights of ``sum(grad_logprob *
        logprob + grad_entropy * entropy)``.  The logits' gradient takes the
        logits' place."""
        entropy = scored.entropy if grad_entropy is not None else None
        g = api.token_logprobs_grad(logits, targets, scored.logsumexp, grad_logprob, entropy, grad_entropy, out=logits)
        return api.matmul_low_f32(g.view(-1, g.shape[-1]).t(), hidden.view(-1, hidden.shape[-1]))

    def generate(self, state: Continuations, tokens: torch.Tensor, steps: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Extends every continuation by ``steps`` tokens, each the likeliest
        one after the last ([G] int32 starts); returns the tokens and their log
        probabilities, [G, steps] each.  ValueError before the first where not
        all of them fit."""
        state.require(tokens.shape[0], steps, self.cfg.positions)
        chosen, scores = [], []
        for _ in range(steps):
            best = api.token_logprobs(self.logits(self.extend(state, tokens[:, None]))[:, 0], top=1)
            tokens = best.top_index[:, 0]
            chosen.append(tokens)
            scores.append(best.top_logprob[:, 0])
        if not chosen:
            return tokens.new_empty(tokens.shape[0], 0), torch.empty(tokens.shape[0], 0, device=tokens.device)
        return torch.stack(chosen, 1), torch.stack(scores, 1)
