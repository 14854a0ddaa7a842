"""A small language model on the selective scan, and its sampled decoding.

Layer stack:

    x -> x + ScanLayer(RMSNorm(x))

ScanLayer: a projection of x to an inner width and a gate of the same; a short
causal convolution with silu (``causal_conv``); the scan's steps (through a
narrow projection), B and C from Linear maps of what comes out; the operator
``selective_scan``, which also applies the gate; the output projection. A
layer's state is the scan's (inner width, states) numbers per sequence and the
convolution's last inputs.

``sample_generate`` prefills a prompt and decodes token by token, the states
updated in place and each token drawn by ``sample_tokens``.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from ramnet_ops import causal_conv, sample_tokens, selective_scan


@dataclass
class ScanConfig:
    vocab: int = 32000
    layers: int = 24
    d_model: int = 1024
    inner: int = 2048
    states: int = 16
    groups: int = 1          # of channels that share B and C
    step_rank: int = 64      # width on the way to the steps
    conv_width: int = 4
    norm_eps: float = 1e-6


class ScanLayer(nn.Module):
    """The operators' caller."""

    def __init__(self, cfg: ScanConfig):
        super().__init__()
        if cfg.inner % cfg.groups:
            raise ValueError(f"inner ({cfg.inner}) must be a multiple of groups ({cfg.groups})")
        self.cfg = cfg
        self.up = nn.Linear(cfg.d_model, 2 * cfg.inner, bias=False)
        self.conv = nn.Parameter(torch.zeros(cfg.inner, cfg.conv_width))
        self.conv_bias = nn.Parameter(torch.zeros(cfg.inner))
        self.mix = nn.Linear(cfg.inner, cfg.step_rank + 2 * cfg.groups * cfg.states, bias=False)
        self.step = nn.Linear(cfg.step_rank, cfg.inner, bias=False)
        self.step_bias = nn.Parameter(torch.zeros(cfg.inner))
        self.log_rate = nn.Parameter(torch.zeros(cfg.inner, cfg.states))
        self.skip = nn.Parameter(torch.ones(cfg.inner))
        self.out = nn.Linear(cfg.inner, cfg.d_model, bias=False)

    @torch.no_grad()
    def init_weights(self, std: float = 0.02) -> None:
        c = self.cfg
        for lin in (self.up, self.mix, self.out):
            nn.init.normal_(lin.weight, 0.0, std)
        nn.init.uniform_(self.step.weight, -c.step_rank ** -0.5, c.step_rank ** -0.5)
        nn.init.uniform_(self.conv, -c.conv_width ** -0.5, c.conv_width ** -0.5)
        nn.init.zeros_(self.conv_bias)
        # steps of 0.001 to 0.1 over the channels (through the softplus), rates of 1, 2, ... over the states
        step = torch.logspace(-3, -1, c.inner, device=self.step_bias.device)
        self.step_bias.copy_(step + torch.log(-torch.expm1(-step)))
        self.log_rate.copy_(torch.log(torch.arange(1, c.states + 1, device=self.log_rate.device).float()).expand(c.inner, -1))
        nn.init.ones_(self.skip)

    def forward(self, x, state, lengths=None, inplace: bool = False):
        c = self.cfg
        h, tail = state
        u, gate = self.up(x).chunk(2, dim=-1)
        u, tail = causal_conv(u, self.conv, self.conv_bias, activation="silu", init_state=tail, lengths=lengths,
                              inplace=inplace)
        step, B, C = self.mix(u).split((c.step_rank, c.groups * c.states, c.groups * c.states), dim=-1)
        y, h = selective_scan(u, self.step(step), -torch.exp(self.log_rate.float()), B.unflatten(-1, (c.groups, c.states)),
                              C.unflatten(-1, (c.groups, c.states)), skip=self.skip, gate=gate, dt_bias=self.step_bias,
                              softplus=True, init_state=h, lengths=lengths, inplace=inplace)
        return self.out(y), (h, tail)


class ScanLM(nn.Module):
    def __init__(self, cfg: ScanConfig):
        super().__init__()
        self.cfg = cfg
        self.embed = nn.Embedding(cfg.vocab, cfg.d_model)
        self.norms = nn.ModuleList(nn.RMSNorm(cfg.d_model, eps=cfg.norm_eps) for _ in range(cfg.layers))
        self.layers = nn.ModuleList(ScanLayer(cfg) for _ in range(cfg.layers))
        self.norm = nn.RMSNorm(cfg.d_model, eps=cfg.norm_eps)
        self.head = nn.Linear(cfg.d_model, cfg.vocab, bias=False)

    @torch.no_grad()
    def init_weights(self, std: float = 0.02) -> None:
        nn.init.normal_(self.embed.weight, 0.0, std)
        nn.init.normal_(self.head.weight, 0.0, std)
        for layer in self.layers:
            layer.init_weights(std)

    def fresh_state(self, batch: int, device) -> list:
        """Per layer the scan's states and the convolution's last inputs: zeros."""
        c = self.cfg
        return [(torch.zeros(batch, c.inner, c.states, device=device),
                 layer.conv.new_zeros(batch, c.conv_width - 1, c.inner, device=device)) for layer in self.layers]

    def forward(self, tokens: torch.Tensor, states: list, lengths=None, inplace: bool = False):
        """Logits (B, T, vocab) and the states. `lengths` (B): the tokens of each row that move its states."""
        x = self.embed(tokens)
        out_states = []
        for norm, layer, st in zip(self.norms, self.layers, states):
            h, st = layer(norm(x), st, lengths, inplace)
            x = x + h
            out_states.append(st)
        return self.head(self.norm(x)), out_states


@torch.no_grad()
def sample_generate(model: ScanLM, prompt: torch.Tensor, new_tokens: int, lengths: torch.Tensor | None = None,
                    temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor | None = None,
                    top_p: float | torch.Tensor | None = None, min_p: float | torch.Tensor | None = None,
                    generator: torch.Generator | None = None):
    """Sample `new_tokens` tokens after each row of ``prompt`` (B, T), padded behind `lengths` (B, at least 1).
    Settings are numbers, or tensors of one value a row (B). Returns the tokens (B, new_tokens) and the states after
    the prompt and all of them but the last."""
    if new_tokens < 1:
        raise ValueError(f"new_tokens must be at least 1, got {new_tokens}")
    B, dev = prompt.shape[0], prompt.device
    settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    logits, states = model(prompt, model.fresh_state(B, dev), lengths)
    if lengths is None:
        logits = logits[:, -1]
    else:
        logits = logits[torch.arange(B, device=dev), lengths.long() - 1]
    out = []
    for step in range(new_tokens):
        token = sample_tokens(logits, torch.rand(B, device=dev, generator=generator), **settings)
        out.append(token)
        if step + 1 < new_tokens:
            logits, states = model(token.unsqueeze(1), states, inplace=True)
            logits = logits[:, -1]
    return torch.stack(out, dim=1), states
