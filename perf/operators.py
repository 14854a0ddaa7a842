"""Timed cases of the gated delta rule and of the verification of drafted tokens.

A case is a plain dict; ``prepare`` makes its inputs on the GPU, ``run`` makes
one pass, through the entry points of ``ramnet_ops`` where ``own`` is set and
through elementary torch operations elsewhere, ``exact`` restates the gated
delta rule in 64 bits, token by token.

The gated delta rule keeps one matrix S (Dk x Dv, 32 bits) per head:

    S <- exp(g_t) S;  u = beta_t (v_t - S^T k_t);  S <- S + k_t u^T
    o_t = scale * S^T q_t

Tensors are laid out as a model's projections give them: q, k (B, T, Hk, Dk),
v (B, T, Hv, Dv), g, beta (B, T, Hv), the state (B, Hv, Dk, Dv). Each q/k head
serves Hv / Hk consecutive heads of v. Packed sequences lie one after the other
in a batch of one, cut by ``cu_seqlens``.

Kinds of case:
  prompt   gated_delta_rule over whole sequences, no gradients
  train    the same with gradients of every input: forward and backward
  step     the tokens of one decode step (one, or a few drafted ones)
  verify   verify_drafts: drafted tokens against the target's probabilities
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ram-net_amd")
_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_CHUNK = 64


def _delta(name, kind, B, T, Hk, Hv, Dk, Dv, dtype, packed=0, state=True, gates="fp32", lengths=False):
    """B sequences of T tokens, or `packed` sequences of T tokens in all."""
    return dict(name=name, kind=kind, B=B, T=T, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype=dtype, packed=packed, state=state,
                gates=gates, lengths=lengths)


def _verify(name, B, S, V, dtype, drafts=True, ragged=False):
    """B sequences with up to S drafted tokens over a vocabulary of V."""
    return dict(name=name, kind="verify", B=B, S=S, V=V, dtype=dtype, drafts=drafts, ragged=ragged)


def listed():
    return [
        # one short prompt on the heads of a small model: launches and latency
        _delta("prompt_short", "prompt", 1, 37, 4, 4, 64, 64, "bf16", state=False),
        # eight 4096-token prompts, the main prefill's heads: the throughput case
        _delta("prompt_batch", "prompt", 8, 4096, 16, 16, 128, 128, "bf16"),
        # one long document on the language model's heads: little but the time axis to work along
        _delta("prompt_long", "prompt", 1, 32768, 8, 8, 128, 128, "bf16", state=False),
        # requests of unequal lengths packed by a server, an empty and a one-token one among them,
        # two value heads to a key head, live states
        _delta("prompt_packed", "prompt", 1, 12345, 8, 16, 128, 128, "fp16", packed=13, gates="same"),
        # a training step of a hybrid model's layer
        _delta("train_batch", "train", 4, 2048, 8, 8, 128, 128, "bf16", state=False),
        # truncated back-propagation over packed documents: shared key heads, odd head sizes, the state's gradient too
        _delta("train_packed", "train", 1, 3001, 3, 6, 72, 96, "fp32", packed=5),
        # one user's next token, the smallest call there is
        _delta("step_single", "step", 1, 1, 8, 8, 128, 128, "bf16"),
        # batch decode, the decode benchmark's heads
        _delta("step_batch", "step", 64, 1, 16, 16, 128, 128, "bf16"),
        # up to six drafted tokens for each of 32 sequences in one call
        _delta("step_drafted", "step", 32, 6, 8, 16, 128, 128, "bf16", lengths=True),
        # one user's three drafted tokens over the language model's vocabulary
        _verify("verify_single", 1, 3, 32000, "fp32"),
        # a serving batch whose drafts come with no probabilities (looked up in the prompt), half-width probabilities
        _verify("verify_lookup", 48, 5, 32000, "bf16", drafts=False, ragged=True),
        # the largest batch and a large odd vocabulary
        _verify("verify_batch", 192, 4, 128257, "fp32", ragged=True),
    ]


def draw(rng):
    """One more case of the same ranges, no dearer than the largest listed one."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["prompt", "prompt", "train", "train", "step", "step", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "verify":
        B, S, V = spread(1, 192), rng.randint(1, 8), spread(1000, 130000)
        while B * S * V > 192 * 4 * 128257:
            B //= 2
        case = _verify("", B, S, V, dtype, drafts=rng.random() < 0.75, ragged=rng.random() < 0.5)
        del case["name"]
        return case
    Hk, group = rng.choice([1, 4, 8, rng.randint(1, 12)]), rng.choice([1, 1, 2, 3])
    Dk = rng.choice([64, 128, 128, 8 * rng.randint(4, 20), rng.randint(20, 160)])
    Dv = rng.choice([Dk, 64, 128, 8 * rng.randint(4, 32), rng.randint(20, 200)])
    more = dict(state=rng.random() < 0.6, gates=rng.choice(["fp32", "same"]))
    if kind == "step":
        B, T = spread(1, 96), rng.choice([1, 1, rng.randint(2, 12)])
        while B > 1 and B * Hk * group * Dk * Dv > 64 * 16 * 128 * 128:
            B //= 2
        case = _delta("", kind, B, T, Hk, Hk * group, Dk, Dv, dtype, lengths=T > 1 and rng.random() < 0.5, **more)
    else:
        T, B = spread(1, 16384), 1
        packed = rng.choice([0, 0, rng.randint(1, 16)])
        most = 8 * 16 * 4096 * 128 * 128 // (8 if kind == "train" else 2) // (4 if dtype == "fp32" else 1)
        if not packed:
            B = spread(1, 12)
        while B > 1 and B * T * Hk * group * Dk * Dv > most:
            B //= 2
        while B * T * Hk * group * Dk * Dv > most:
            T //= 2
        case = _delta("", kind, B, T, Hk, Hk * group, Dk, Dv, dtype, packed=packed, **more)
    del case["name"]
    return case


# --------------------------------------------------------------------------
# inputs

def _lens(case, seed):
    """Lengths of the packed sequences: an empty and a one-token one among four or more."""
    N, T, r = case["packed"], case["T"], random.Random(seed)
    fixed = [0, 1] if N >= 4 and T > N else []
    cuts = sorted(r.randint(0, T - sum(fixed)) for _ in range(N - len(fixed) - 1))
    lens = [b - a for a, b in zip([0] + cuts, cuts + [T - sum(fixed)])]
    for n in fixed:
        lens.insert(r.randint(0, len(lens)), n)
    return lens


def _prepare_verify(case, gen):
    B, S, V, dtype = case["B"], case["S"], case["V"], _DTYPES[case["dtype"]]
    dev = "cuda"
    logits = torch.randn(B, S + 1, V, generator=gen, device=dev).mul_(2.0)
    target = torch.softmax(logits, -1).to(dtype)
    # the draft model's view of the same logits: near the target, so that most drafts are taken
    near = logits[:, :S].add_(torch.randn(B, S, V, generator=gen, device=dev), alpha=0.5)
    draft = torch.softmax(near, -1)
    del logits, near
    tokens = torch.multinomial(draft.view(B * S, V), 1, generator=gen).view(B, S)
    lens = torch.randint(0, S + 1, (B,), generator=gen, device=dev, dtype=torch.int32) if case["ragged"] else None
    return dict(case=case, tokens=tokens, target=target, draft=draft.to(dtype) if case["drafts"] else None,
                accept=torch.rand(B, S, generator=gen, device=dev), sample=torch.rand(B, generator=gen, device=dev),
                lens=lens)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "verify":
        return _prepare_verify(case, gen)
    B, T, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    dtype = _DTYPES[case["dtype"]]
    gate_type = torch.float32 if case["gates"] == "fp32" else dtype

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    # unit keys and queries, as the layer normalises them; decays and write strengths as its gates give them:
    # rates from 1 to 16 a step of 0.001 to 0.1, and half of the strength on average
    q = torch.nn.functional.normalize(randn(B, T, Hk, Dk), dim=-1).to(dtype)
    k = torch.nn.functional.normalize(randn(B, T, Hk, Dk), dim=-1).to(dtype)
    v = randn(B, T, Hv, Dv).to(dtype)
    rate = torch.rand(Hv, generator=gen, device="cuda") * 15 + 1
    bias = torch.exp(torch.rand(Hv, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    bias = bias + torch.log(-torch.expm1(-bias))
    g = (-rate * torch.nn.functional.softplus(0.5 * randn(B, T, Hv) + bias)).to(gate_type)
    beta = torch.sigmoid(randn(B, T, Hv)).to(dtype)
    N = case["packed"] or B
    init = 0.3 * randn(N, Hv, Dk, Dv) if case["state"] else None
    state = dict(case=case, q=q, k=k, v=v, g=g, beta=beta, init=init, cu=None, max_len=T, lengths=None)
    if case["packed"]:
        lens = _lens(case, seed)
        state["cu"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        state["max_len"] = max(lens)
    if case["lengths"]:
        state["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    if case["kind"] == "train":
        state["do"] = randn(B, T, Hv, Dv).to(dtype)
        state["dstate"] = 0.3 * randn(N, Hv, Dk, Dv)
    return state


# --------------------------------------------------------------------------
# plain forms

def _unpack(x, cu, max_len):
    """(1, T, ...) packed to (N, max_len, ...), zeros after each sequence's end."""
    at = cu[:-1, None].long() + torch.arange(max_len, device=x.device)
    out = x[0][at.clamp(max=x.shape[1] - 1)]
    return out.masked_fill((at >= cu[1:, None]).view(*at.shape, *[1] * (x.dim() - 2)), 0)


def _pack(x, cu, T):
    """The other way: (N, max_len, ...) to (1, T, ...)."""
    token = torch.arange(T, device=x.device)
    n = torch.searchsorted(cu[1:].contiguous(), token.to(cu.dtype), right=True)
    return x[n, token - cu[n].long()].unsqueeze(0)


def _inverse(m):
    """Inverse of unit lower triangular matrices, in blocks of twice the size each turn."""
    n = m.shape[-1]
    x = torch.ones(*m.shape[:-1], 1, device=m.device, dtype=m.dtype).unsqueeze(-2)  # (..., n, 1, 1)
    s = 1
    while s < n:
        blocks = m.unflatten(-1, (n // (2 * s), 2 * s)).unflatten(-3, (n // (2 * s), 2 * s))
        low = torch.diagonal(blocks, dim1=-4, dim2=-2).movedim(-1, -3)[..., s:, :s]
        a, b = x[..., 0::2, :, :], x[..., 1::2, :, :]
        low = -(b @ low.contiguous() @ a)
        x = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([low, b], -1)], -2)
        s *= 2
    return x.squeeze(-3)


def _chunked(q, k, v, g, beta, state, scale):
    """The rule in chunks of 64 tokens: products over a chunk, a loop over chunks. (N, T, H, D) in 32 bits."""
    N, T, Hk, Dk = k.shape
    Hv, Dv = v.shape[2:]
    c = -(-T // _CHUNK)

    def chunks(x):
        x = torch.nn.functional.pad(x, (0,) * (2 * (x.dim() - 2)) + (0, c * _CHUNK - T))
        if x.shape[2] != Hv:
            x = x.repeat_interleave(Hv // Hk, 2)
        return x.transpose(1, 2).unflatten(2, (c, _CHUNK)).contiguous()  # (N, H, c, 64, ...)

    q, k, v, beta = chunks(q), chunks(k), chunks(v), chunks(beta)
    gam = chunks(g).double().cumsum(-1)
    upper = torch.ones(_CHUNK, _CHUNK, device=q.device, dtype=torch.bool).triu(1)
    decay = (gam.unsqueeze(-1) - gam.unsqueeze(-2)).masked_fill(upper, -math.inf).exp().float()
    kt = k.transpose(-1, -2).contiguous()
    mix = beta.unsqueeze(-1) * ((k @ kt) * decay).tril(-1) + torch.eye(_CHUNK, device=q.device)
    inv, p = _inverse(mix), (q @ kt) * decay
    grow, left = gam.exp().float().unsqueeze(-1), (gam[..., -1:] - gam).exp().float().unsqueeze(-1)
    total = gam[..., -1].exp().float()[..., None, None]
    bv, bk, qg, kl = beta.unsqueeze(-1) * v, beta.unsqueeze(-1) * grow * k, grow * q, (left * k).transpose(-1, -2)
    kl = kl.contiguous()
    o = []
    for i in range(c):
        u = inv[:, :, i] @ (bv[:, :, i] - bk[:, :, i] @ state)
        o.append(qg[:, :, i] @ state + p[:, :, i] @ u)
        state = total[:, :, i] * state + kl[:, :, i] @ u
    o = scale * torch.cat(o, 2)
    return o[:, :, :T].transpose(1, 2), state


def _plain_rule(s, q, k, v, g, beta, init):
    case, cu = s["case"], s["cu"]
    T, Hv, Dk, Dv = case["T"], case["Hv"], case["Dk"], case["Dv"]
    args = [x.float() for x in (q, k, v, g, beta)]
    N = case["packed"] or case["B"]
    if init is None:
        init = torch.zeros(N, Hv, Dk, Dv, device=q.device)
    if cu is not None:
        args = [_unpack(x, cu, s["max_len"]) for x in args]
    o, state = _chunked(*args, init, case["Dk"] ** -0.5)
    if cu is not None:
        o = _pack(o, cu, T)
    return o.to(v.dtype), state


def _plain_step(s):
    """Token by token, as few as there are."""
    case = s["case"]
    Hk, Hv, Dk, Dv, T = (case[n] for n in ("Hk", "Hv", "Dk", "Dv", "T"))
    q, k = (s[n].float().repeat_interleave(Hv // Hk, 2) for n in "qk")
    v, g, beta = s["v"].float(), s["g"].float(), s["beta"].float()
    state = s["init"]
    if state is None:
        state = torch.zeros(case["B"], Hv, Dk, Dv, device=q.device)
    o = []
    for t in range(T):
        old = state
        state = g[:, t, :, None, None].exp() * state
        kt = k[:, t].unsqueeze(-1)
        u = beta[:, t].unsqueeze(-1) * (v[:, t] - (state * kt).sum(-2))
        state = state + kt * u.unsqueeze(-2)
        out = (state * q[:, t].unsqueeze(-1)).sum(-2) * Dk ** -0.5
        if s["lengths"] is not None:
            live = (t < s["lengths"]).view(-1, 1, 1)
            out = torch.where(live, out, 0.0)
            state = torch.where(live.unsqueeze(-1), state, old)
        o.append(out)
    return torch.stack(o, 1).to(s["v"].dtype), state


def _plain_verify(s):
    tokens, target, draft, lens = s["tokens"], s["target"], s["draft"], s["lens"]
    B, S = tokens.shape
    dev = tokens.device
    if lens is None:
        lens = torch.full((B,), S, device=dev)
    at = tokens.unsqueeze(-1)
    p = target[:, :S].gather(-1, at).squeeze(-1).double()
    q = draft.gather(-1, at).squeeze(-1).double() if draft is not None else torch.ones_like(p)
    step = torch.arange(S, device=dev)
    taken = (s["accept"].double() * q < p) & (step < lens.unsqueeze(-1))
    n = taken.long().cumprod(-1).sum(-1)
    row = torch.arange(B, device=dev)
    weight = target[row, n].double()
    last = n.clamp(max=S - 1)
    if draft is not None:
        other = draft[row, last].double()
    else:
        other = torch.zeros_like(weight).scatter(-1, tokens[row, last].unsqueeze(-1), math.inf)
    refused = (n < lens).unsqueeze(-1)
    rest = (weight - torch.where(refused, other, 0.0)).clamp(min=0)
    weight = torch.where(rest.sum(-1, keepdim=True) > 0, rest, weight)
    total = weight.cumsum(-1)
    over = (total > s["sample"].double().unsqueeze(-1) * total[:, -1:]) & (weight > 0)
    chosen = over.long().argmax(-1)
    out = torch.where(step < n.unsqueeze(-1), tokens, -1)
    out = torch.cat([out, torch.full((B, 1), -1, device=dev)], 1).scatter(1, n.unsqueeze(-1), chosen.unsqueeze(-1))
    return out, n.to(torch.int32)


# --------------------------------------------------------------------------
# one pass

_INPUTS = ("q", "k", "v", "g", "beta", "init")


def _own_rule(s, q, k, v, g, beta, init):
    from ramnet_ops import gated_delta_rule
    return gated_delta_rule(q, k, v, g, beta, init_state=init, cu_seqlens=s["cu"], lengths=s["lengths"])


def _own_verify(s):
    from ramnet_ops import verify_drafts
    return verify_drafts(s["tokens"], s["target"], s["draft"], s["accept"], s["sample"], draft_lens=s["lens"])


def _train(rule, s):
    names = [n for n in _INPUTS if s[n] is not None]
    leaves = {n: s[n].detach().requires_grad_() for n in names}
    o, state = rule(s, *(leaves.get(n) for n in _INPUTS))
    grads = torch.autograd.grad([o, state], [leaves[n] for n in names], [s["do"], s["dstate"]])
    return {"o": o.detach(), "state": state.detach(), **{"d" + n: d for n, d in zip(names, grads)}}


def run(state):
    kind = state["case"]["kind"]
    if own and _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    if kind == "verify":
        tokens, taken = _own_verify(state) if own else _plain_verify(state)
        return {"tokens": tokens, "taken": taken}
    rule = _own_rule if own else _plain_rule
    if kind == "train":
        return _train(rule, state)
    with torch.no_grad():
        if kind == "step" and not own:
            o, new = _plain_step(state)
        else:
            o, new = rule(state, *(state[n] for n in _INPUTS))
    return {"o": o, "state": new}


# --------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "verify":
        # one target row and one draft row of each sequence are read whole
        B, S, V = case["B"], case["S"], case["V"]
        rows = 2 if case["drafts"] else 1
        return {"bytes": B * V * size * rows + B * S * (8 + 4 + 2 * size) + B * (S + 1) * 8 + B * 8, "flops": 4 * B * V}
    B, T, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
    gate = (4 if case["gates"] == "fp32" else size) + size
    token = 2 * Hk * Dk * size + Hv * Dv * size + Hv * gate
    matrix = (case["packed"] or B) * Hv * Dk * Dv * 4
    data = B * T * (token + Hv * Dv * size) + matrix * (2 if case["state"] else 1)
    # S^T k, k u^T and S^T q of each token
    flops = 6 * B * T * Hv * Dk * Dv
    if case["kind"] == "train":
        # the inputs once more with the output's gradient, and every gradient written
        data += B * T * (2 * token + Hv * Dv * size) + matrix * (2 if case["state"] else 1)
        flops *= 3
    return {"bytes": data, "flops": flops}


# --------------------------------------------------------------------------
# 64 bits

def _segments(case, seed, s):
    """Inputs in 64 bits as (N, L, ...), one row a sequence, and how many of its tokens count."""
    q, k, v, g, beta = (s[n].double() for n in _INPUTS[:5])
    if case["packed"]:
        lens = _lens(case, seed)
        rows = []
        for x in (q, k, v, g, beta):
            parts = x[0].split(lens)
            rows.append(torch.nn.utils.rnn.pad_sequence(parts, batch_first=True))
        q, k, v, g, beta = rows
    elif case["lengths"]:
        lens = s["lengths"].tolist()
    else:
        lens = [case["T"]] * case["B"]
    live = torch.arange(q.shape[1], device=q.device) < torch.tensor(lens, device=q.device).unsqueeze(-1)
    # a token that does not count neither decays nor writes
    g, beta = g * live.unsqueeze(-1), beta * live.unsqueeze(-1)
    group = case["Hv"] // case["Hk"]
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    return q, k, v, g, beta, lens, live


def _join(case, x, lens):
    """Back to the layout of the inputs, without the padding."""
    if case["packed"]:
        return torch.cat([row[:n] for row, n in zip(x, lens)]).unsqueeze(0)
    return x


def _walk(k, v, alpha, beta, S, each):
    """The states from S on over the tokens of (N, L, H, D) inputs; each(t, decayed, error, after)."""
    for t in range(k.shape[1]):
        decayed = alpha[:, t, :, None, None] * S
        error = v[:, t] - (decayed * k[:, t].unsqueeze(-1)).sum(-2)
        S = decayed + k[:, t].unsqueeze(-1) * (beta[:, t].unsqueeze(-1) * error).unsqueeze(-2)
        each(t, decayed, error, S)
    return S


def exact(case, seed):
    """The outputs of one pass in 64 bits: the recurrence token by token, and its adjoint backwards.
    The tokens and counts of a verification are whole numbers, which have to be equal: no values here."""
    if case["kind"] == "verify":
        return None
    s = prepare(case, seed)
    q, k, v, g, beta, lens, live = _segments(case, seed, s)
    alpha = g.exp()
    N, L, Hv, Dk = q.shape
    Dv, scale = case["Dv"], Dk ** -0.5
    S = s["init"].double() if s["init"] is not None else torch.zeros(N, Hv, Dk, Dv, device=q.device).double()
    o = torch.zeros(N, L, Hv, Dv, device=q.device, dtype=torch.float64)
    at, span = [], 32  # the state before every `span` tokens, to walk forward from again

    def read(t, decayed, error, after):
        o[:, t] = scale * (after * q[:, t].unsqueeze(-1)).sum(-2)

    for t in range(0, L, span):
        cut = slice(t, t + span)
        at.append(S if case["kind"] == "train" else None)
        S = _walk(k[:, cut], v[:, cut], alpha[:, cut], beta[:, cut], S, lambda i, *x, t=t: read(t + i, *x))
    o = o * live[:, :, None, None]
    out = {"o": _join(case, o, lens), "state": S}
    if case["kind"] != "train":
        return out

    do = s["do"].double()
    if case["packed"]:
        do = torch.nn.utils.rnn.pad_sequence(do[0].split(lens), batch_first=True)
    dq, dk, dv, dg, dbeta = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    D = s["dstate"].double()
    for t in reversed(range(0, L, span)):
        cut, seen = slice(t, t + span), []
        _walk(k[:, cut], v[:, cut], alpha[:, cut], beta[:, cut], at[t // span], lambda i, *x: seen.append(x))
        for i in reversed(range(len(seen))):
            j, (decayed, error, after) = t + i, seen[i]
            kj, bj = k[:, j].unsqueeze(-1), beta[:, j].unsqueeze(-1)
            dq[:, j] = scale * (after * do[:, j].unsqueeze(-2)).sum(-1)
            D = D + scale * q[:, j].unsqueeze(-1) * do[:, j].unsqueeze(-2)
            du = (D * kj).sum(-2)
            dbeta[:, j] = (du * error).sum(-1)
            dv[:, j] = bj * du
            dk[:, j] = (D * (bj * error).unsqueeze(-2)).sum(-1) - (decayed * dv[:, j].unsqueeze(-2)).sum(-1)
            D = D - kj * dv[:, j].unsqueeze(-2)
            dg[:, j] = (D * decayed).sum((-1, -2))
            D = alpha[:, j, :, None, None] * D
    shared = (N, L, case["Hk"], Hv // case["Hk"], Dk)
    dq, dk = dq.view(shared).sum(3), dk.view(shared).sum(3)
    out.update({n: _join(case, x, lens) for n, x in (("dq", dq), ("dk", dk), ("dv", dv), ("dg", dg), ("dbeta", dbeta))})
    if s["init"] is not None:
        out["dinit"] = D
    return out
