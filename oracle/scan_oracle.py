"""fp64 restatements of the short causal convolution, the selective scan and token sampling.

Token by token and row by row, from the definitions; differentiable (autograd)
where the operator is. No code of the package is used.
"""
from __future__ import annotations

import math

import torch


def spans_of(B, T, lens, packed):
    """(row, first token, length) of each sequence."""
    if lens is None:
        lens = [T] * B
    out, start = [], 0
    for n, length in enumerate(lens):
        out.append((0, start, length) if packed else (n, 0, length))
        start += length
    return out


def causal_conv(x, weight, bias=None, silu=False, init_state=None, lens=None, packed=False):
    """(y, state) in float64. ``lens``: tokens of each row that count, or (packed) of each of
    the sequences that follow one another in the one row."""
    x, weight = x.double(), weight.double()
    B, T, D = x.shape
    W = weight.shape[1]
    rows, states = {}, []
    spans = spans_of(B, T, lens, packed)
    for n, (b, t0, length) in enumerate(spans):
        before = x.new_zeros(W - 1, D) if init_state is None else init_state[n].double()
        line = torch.cat([before, x[b, t0:t0 + length]])
        for t in range(length):
            s = (line[t:t + W] * weight.t()).sum(0)
            if bias is not None:
                s = s + bias.double()
            rows[b, t0 + t] = s / (1 + (-s).exp()) if silu else s
        states.append(line[length:])
    zero = x.new_zeros(D)
    y = torch.stack([rows.get((b, t), zero) for b in range(B) for t in range(T)]) if B * T else x.new_zeros(0)
    return y.reshape(B, T, D), torch.stack(states).reshape(len(spans), W - 1, D) if spans else x.new_zeros(0, W - 1, D)


def selective_scan(x, dt, A, B, C, skip=None, gate=None, dt_bias=None, softplus=False, init_state=None, lens=None,
                   packed=False):
    """(y, state) in float64."""
    x, dt, A, B, C = (t.double() for t in (x, dt, A, B, C))
    batch, T, D = x.shape
    S, wide = A.shape[1], D // B.shape[2]
    if dt_bias is not None:
        dt = dt + dt_bias.double()
    if softplus:
        dt = torch.where(dt > 30, dt, dt.clamp(max=30).exp().log1p())
    rows, states = {}, []
    spans = spans_of(batch, T, lens, packed)
    for n, (b, t0, length) in enumerate(spans):
        h = x.new_zeros(D, S) if init_state is None else init_state[n].double()
        for t in range(t0, t0 + length):
            d = dt[b, t].unsqueeze(-1)
            h = (d * A).exp() * h + d * x[b, t].unsqueeze(-1) * B[b, t].repeat_interleave(wide, 0)
            y = (h * C[b, t].repeat_interleave(wide, 0)).sum(-1)
            if skip is not None:
                y = y + skip.double() * x[b, t]
            if gate is not None:
                z = gate[b, t].double()
                y = y * z / (1 + (-z).exp())
            rows[b, t] = y
        states.append(h)
    zero = x.new_zeros(D)
    y = torch.stack([rows.get((b, t), zero) for b in range(batch) for t in range(T)]) if batch * T else x.new_zeros(0)
    return y.reshape(batch, T, D), torch.stack(states) if spans else x.new_zeros(0, D, S)


def sample_row(logits, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probabilities) of one row, by Python's own sort."""
    values = [float(v) for v in logits]
    values = [-math.inf if math.isnan(v) else v for v in values]
    top = max(values)
    probs = torch.zeros(len(values), dtype=torch.float64)
    if top == -math.inf:
        return 0, probs
    greedy = not temperature > 0

    def weight(v):
        if v == top:
            return 1.0
        return 0.0 if v == -math.inf or top == math.inf else math.exp((v - top) / (1.0 if greedy else temperature))
    order = sorted(range(len(values)), key=lambda i: (-values[i], i))
    if greedy:
        order = order[:1]
    elif top_k > 0:
        order = order[:top_k]
    weights = [weight(values[i]) for i in order]
    total, before, kept = math.fsum(weights), 0.0, []
    for place, (i, w) in enumerate(zip(order, weights)):
        if place and (top_p < 1 and not before < top_p * total or w < min(min_p, 1.0)):
            break
        kept.append(i)
        before += w
    kept = [i for i in sorted(kept) if values[i] > -math.inf]
    for i in kept:
        probs[i] = weight(values[i])
    total, run, token = math.fsum(probs.tolist()), 0.0, kept[-1]
    for i in kept:
        run += float(probs[i])
        if run > random * total and probs[i] > 0:
            token = i
            break
    return token, probs / total
