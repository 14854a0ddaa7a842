"""A small language model on the gated delta rule, and its speculative decoding.

Layer stack:

    x -> x + DeltaLayer(RMSNorm(x)) -> x + SwiGLU(RMSNorm(x))

DeltaLayer: queries, keys (each of norm 1), values, a decay and a write
strength per value head from Linear maps of x; where ``conv_width`` is set, a
short causal convolution with silu of the queries, keys and values
(``causal_conv``); the operator ``gated_delta_rule``; a head-wise RMSNorm of what
it reads, a sigmoid gate and the output projection, as RamLayer has them. The
state is the operator's, one (key_dim, value_dim) matrix per sequence and value
head, and with a convolution also its last inputs: a pair of the two.

``speculative_generate`` decodes with a smaller model that drafts: the target
scores all drafts of a sequence in one call, ``verify_drafts`` says which stay,
and the states move over those alone. A matrix state cannot be cut back the way
a cache of tokens can, so the scoring call leaves the states as they are, each
layer keeps its operators' inputs (a few rows), and the operators run over them
once more in place with the number of tokens that stayed. With ``top_k``,
``top_p`` or ``min_p`` both models' tokens come from what these leave of their
distributions (``sample_tokens``, ``token_probabilities``).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from ramnet_ops import causal_conv, gated_delta_rule, sample_tokens, token_probabilities, verify_drafts

from .lm import SwiGLU


@dataclass
class DeltaConfig:
    vocab: int = 32000
    layers: int = 24
    d_model: int = 1024
    key_heads: int = 8
    heads: int = 8           # value heads, a multiple of key_heads
    key_dim: int = 128
    value_dim: int = 128
    mlp_width: int = 2816
    norm_eps: float = 1e-6
    conv_width: int = 0      # taps of the convolution before the operator; 0: none


class DeltaLayer(nn.Module):
    """The operator's caller: projections, gates and the norm of what is read."""

    def __init__(self, cfg: DeltaConfig):
        super().__init__()
        if cfg.heads % cfg.key_heads:
            raise ValueError(f"heads ({cfg.heads}) must be a multiple of key_heads ({cfg.key_heads})")
        self.cfg = cfg
        d, keys, values = cfg.d_model, cfg.key_heads * cfg.key_dim, cfg.heads * cfg.value_dim
        self.qkv = nn.Linear(d, 2 * keys + values, bias=False)
        self.decay = nn.Linear(d, cfg.heads)
        self.beta = nn.Linear(d, cfg.heads)
        self.gate = nn.Linear(d, values)
        self.out = nn.Linear(values, d, bias=False)
        self.out_norm = nn.RMSNorm(cfg.value_dim, eps=cfg.norm_eps)
        if cfg.conv_width:
            self.conv = nn.Parameter(torch.zeros(2 * keys + values, cfg.conv_width))

    @torch.no_grad()
    def init_weights(self, std: float = 0.02) -> None:
        for lin in (self.qkv, self.decay, self.beta, self.gate, self.out):
            nn.init.normal_(lin.weight, 0.0, std)
        # half-lives of 2 to 2000 tokens over the heads: e^g = 2^(-1 / t), g = -softplus(bias)
        rate = 0.6931 / torch.logspace(0.3, 3.3, self.cfg.heads)
        self.decay.bias.copy_(rate.expm1().log())
        nn.init.zeros_(self.beta.bias)
        nn.init.zeros_(self.gate.bias)
        if self.cfg.conv_width:
            nn.init.uniform_(self.conv, -self.cfg.conv_width ** -0.5, self.cfg.conv_width ** -0.5)

    def op_inputs(self, x: torch.Tensor, qkv: torch.Tensor | None = None):
        """(q, k, v, g, beta) in the operator's (B, T, H, ...) layout."""
        B, T, _ = x.shape
        c = self.cfg
        keys = c.key_heads * c.key_dim
        q, k, v = (self.qkv(x) if qkv is None else qkv).split((keys, keys, c.heads * c.value_dim), dim=-1)
        q = F.normalize(q.view(B, T, c.key_heads, c.key_dim), dim=-1)
        k = F.normalize(k.view(B, T, c.key_heads, c.key_dim), dim=-1)
        # (the decay in 32 bits: over long prompts its sum is what counts)
        return q, k, v.view(B, T, c.heads, c.value_dim), -F.softplus(self.decay(x).float()), torch.sigmoid(self.beta(x))

    def forward(self, x, state, lengths=None, inplace: bool = False, keep=None):
        qkv = tail = raw = None
        if self.cfg.conv_width:
            state, tail = state
            raw = self.qkv(x)
            qkv, tail = causal_conv(raw, self.conv, activation="silu", init_state=tail, lengths=lengths, inplace=inplace)
        inputs = self.op_inputs(x, qkv)
        if keep is not None:
            keep.append(inputs if raw is None else (inputs, raw, self.conv))
        y, state = gated_delta_rule(*inputs, init_state=state, lengths=lengths, inplace=inplace)
        if tail is not None:
            state = (state, tail)
        return self.out(torch.sigmoid(self.gate(x)) * self.out_norm(y).flatten(-2)), state


class DeltaBlock(nn.Module):
    def __init__(self, cfg: DeltaConfig):
        super().__init__()
        self.delta_norm = nn.RMSNorm(cfg.d_model, eps=cfg.norm_eps)
        self.delta = DeltaLayer(cfg)
        self.mlp_norm = nn.RMSNorm(cfg.d_model, eps=cfg.norm_eps)
        self.mlp = SwiGLU(cfg.d_model, cfg.mlp_width)

    def forward(self, x, state, lengths=None, inplace: bool = False, keep=None):
        h, state = self.delta(self.delta_norm(x), state, lengths, inplace, keep)
        x = x + h
        return x + self.mlp(self.mlp_norm(x)), state


class DeltaLM(nn.Module):
    def __init__(self, cfg: DeltaConfig):
        super().__init__()
        self.cfg = cfg
        self.embed = nn.Embedding(cfg.vocab, cfg.d_model)
        self.blocks = nn.ModuleList(DeltaBlock(cfg) for _ in range(cfg.layers))
        self.norm = nn.RMSNorm(cfg.d_model, eps=cfg.norm_eps)
        self.head = nn.Linear(cfg.d_model, cfg.vocab, bias=False)

    @torch.no_grad()
    def init_weights(self, std: float = 0.02) -> None:
        nn.init.normal_(self.embed.weight, 0.0, std)
        nn.init.normal_(self.head.weight, 0.0, std)
        for blk in self.blocks:
            blk.delta.init_weights(std)
            nn.init.normal_(blk.mlp.gate_up.weight, 0.0, std)
            nn.init.normal_(blk.mlp.down.weight, 0.0, std)

    def fresh_state(self, batch: int, device) -> list:
        """Zeros of each layer: the operator's matrices, with a convolution in a pair with its last inputs."""
        cfg = self.cfg
        states = [torch.zeros(batch, cfg.heads, cfg.key_dim, cfg.value_dim, device=device) for _ in range(cfg.layers)]
        if not cfg.conv_width:
            return states
        return [(s, blk.delta.conv.new_zeros(batch, cfg.conv_width - 1, blk.delta.conv.shape[0], device=device))
                for s, blk in zip(states, self.blocks)]

    def forward(self, tokens: torch.Tensor, states: list, lengths=None, inplace: bool = False, keep=None):
        """Logits (B, T, vocab) and the states. `lengths` (B): the tokens of
        each row that move its states; `keep`: a list that gets each layer's
        operator inputs, for ``advance``."""
        x = self.embed(tokens)
        out_states = []
        for blk, st in zip(self.blocks, states):
            x, st = blk(x, st, lengths, inplace, keep)
            out_states.append(st)
        return self.head(self.norm(x)), out_states


@torch.no_grad()
def advance(kept: list, states: list, lengths: torch.Tensor) -> None:
    """Move the states, in place, over the first `lengths` tokens of a scoring call."""
    for inputs, state in zip(kept, states):
        if isinstance(state, tuple):
            inputs, raw, taps = inputs
            state, tail = state
            causal_conv(raw, taps, init_state=tail, lengths=lengths, inplace=True)
        gated_delta_rule(*inputs, init_state=state, lengths=lengths, inplace=True)


def _probabilities(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    return torch.softmax(logits.float() / temperature, dim=-1)


@torch.no_grad()
def speculative_generate(model: DeltaLM, drafter: DeltaLM, prompt: torch.Tensor, new_tokens: int, drafts: int = 4,
                         temperature: float = 1.0, generator: torch.Generator | None = None, top_k: int | None = None,
                         top_p: float | None = None, min_p: float | None = None):
    """Sample `new_tokens` tokens after ``prompt`` (B, T), with up to `drafts`
    of them a step proposed by `drafter`; they are distributed as `model`'s own,
    with what `top_k`, `top_p` and `min_p` leave of it.

    Rows advance by different counts: a row that is done has no drafts and its
    states stay. Returns the tokens (B, new_tokens), the model's states
    after the prompt and all of them but the last, and the number of steps."""
    if drafts < 1:
        raise ValueError(f"drafts must be at least 1, got {drafts}")
    B, dev = prompt.shape[0], prompt.device
    settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    filtered = any(v is not None for v in (top_k, top_p, min_p))

    def probabilities(logits):
        return token_probabilities(logits, **settings) if filtered else _probabilities(logits, temperature)

    def draw(logits):
        """(token (B, 1), probabilities (B, vocab))."""
        if filtered:
            token, chances = sample_tokens(logits, torch.rand(B, device=dev, generator=generator), **settings,
                                           probabilities=True)
            return token.unsqueeze(1), chances
        chances = _probabilities(logits, temperature)
        return torch.multinomial(chances, 1, generator=generator), chances

    logits, states = model(prompt, model.fresh_state(B, dev))
    _, drafter_states = drafter(prompt, drafter.fresh_state(B, dev))
    last, _ = draw(logits[:, -1])
    # one column more, for what a row does not write
    out = torch.empty(B, new_tokens + 1, dtype=torch.long, device=dev)
    out[:, :1] = last
    count = torch.ones(B, 1, dtype=torch.long, device=dev)
    places = torch.arange(drafts + 1, device=dev)
    steps = 0
    while int(count.min()) < new_tokens:
        left = new_tokens - count
        # the drafts, from states that are dropped
        tokens, chances, tried = [last], [], drafter_states
        for _ in range(drafts):
            logits, tried = drafter(tokens[-1], tried)
            token, chance = draw(logits[:, -1])
            tokens.append(token)
            chances.append(chance)
        block = torch.cat(tokens, dim=1)
        # all of them scored in one call, from states that stay
        kept = []
        logits, _ = model(block, states, keep=kept)
        drawn, taken = verify_drafts(
            block[:, 1:], probabilities(logits), torch.stack(chances, dim=1),
            torch.rand(B, drafts, device=dev, generator=generator), torch.rand(B, device=dev, generator=generator),
            draft_lens=(left - 1).clamp(0, drafts).view(B).int())
        taken = taken.view(B, 1)
        moved = torch.where(left > 0, taken + 1, 0)
        lengths = moved.view(B).int()
        advance(kept, states, lengths)
        drafter(block, drafter_states, lengths=lengths, inplace=True)
        out.scatter_(1, torch.where(places < moved, count + places, new_tokens), drawn)
        last = torch.where(left > 0, drawn.gather(1, taken.long()), last)
        count = count + moved
        steps += 1
    return out[:, :new_tokens], states, steps
