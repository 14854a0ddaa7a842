"""fp64 restatements of the gated delta rule and of draft verification.

Token by token and row by row, from the definitions; differentiable (autograd)
where the operator is. No code of the package is used.
"""
from __future__ import annotations

import torch


def delta_rule(q, k, v, g, beta, scale=None, init_state=None, lens=None, packed=False):
    """(o, state) in float64. ``lens``: tokens of each row that count, or (packed)
    of each of the sequences that follow one another in the one row."""
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    scale = Dk ** -0.5 if scale is None else scale
    q, k = (t.repeat_interleave(Hv // Hk, 2) for t in (q, k))
    if lens is None:
        lens = [T] * B
    spans = []
    start = 0
    for n, length in enumerate(lens):
        spans.append((0, start, length) if packed else (n, 0, length))
        start += length
    rows = {}
    states = []
    for n, (b, t0, length) in enumerate(spans):
        S = torch.zeros(Hv, Dk, Dv, dtype=torch.float64) if init_state is None else init_state[n].double()
        for t in range(t0, t0 + length):
            S = g[b, t].exp()[:, None, None] * S
            u = beta[b, t][:, None] * (v[b, t] - torch.einsum("hkv,hk->hv", S, k[b, t]))
            S = S + k[b, t].unsqueeze(-1) * u.unsqueeze(-2)
            rows[b, t] = scale * torch.einsum("hkv,hk->hv", S, q[b, t])
        states.append(S)
    zero = torch.zeros(Hv, Dv, dtype=torch.float64)
    o = torch.stack([rows.get((b, t), zero) for b in range(B) for t in range(T)]) if B * T else torch.zeros(0)
    state = torch.stack(states) if states else torch.zeros(0)
    return o.reshape(B, T, Hv, Dv), state.reshape(len(spans), Hv, Dk, Dv)


def verify_drafts(tokens, target, draft, accept, sample, lens=None):
    """(tokens, taken), one row after the other in float64."""
    B, S = tokens.shape
    V = target.shape[2]
    out = torch.full((B, S + 1), -1, dtype=torch.int64)
    taken = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n, length = 0, S if lens is None else int(lens[b])
        while n < length:
            x = int(tokens[b, n])
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else float(draft[b, n, x])
            if not float(accept[b, n]) * q < float(target[b, n, x]):
                break
            out[b, n] = x
            n += 1
        p = target[b, n].double()
        rest = p
        if n < length and draft is not None:
            rest = (p - draft[b, n].double()).clamp(min=0)
        elif n < length:
            rest = p.clone()
            if 0 <= int(tokens[b, n]) < V:
                rest[int(tokens[b, n])] = 0
        if not float(rest.sum()) > 0:
            rest = p
        run = rest.cumsum(0)
        over = ((run > float(sample[b]) * run[-1]) & (rest > 0)).nonzero()
        out[b, n] = int(over[0]) if len(over) else 0
        taken[b] = n
    return out, taken
