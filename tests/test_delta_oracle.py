"""The fp64 oracle of the gated delta rule and of draft verification against
closed forms, and its gradient against differences (CPU)."""
from __future__ import annotations

import pytest
import torch

from oracle import delta_oracle as oracle


def _inputs(B=1, T=6, Hk=1, Hv=2, Dk=3, Dv=4, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)
    k = torch.nn.functional.normalize(rn(B, T, Hk, Dk), dim=-1)
    return [rn(B, T, Hk, Dk), k, rn(B, T, Hv, Dv), -rn(B, T, Hv).abs(), torch.sigmoid(rn(B, T, Hv)),
            rn(B, Hv, Dk, Dv)]


def test_without_gates_it_is_an_overwriting_memory():
    # orthonormal keys, beta = 1, no decay: reading key i gives the last value written at it
    T, D = 5, 5
    k = torch.eye(D, dtype=torch.float64).view(1, T, 1, D)
    v = torch.randn(1, T, 1, 3, dtype=torch.float64)
    zero, one = torch.zeros(1, T, 1), torch.ones(1, T, 1)
    o, state = oracle.delta_rule(k, k, v, zero, one, scale=1.0)
    assert torch.allclose(o, v) and torch.allclose(state[0, 0], v[0, :, 0])
    again = torch.cat([k, k], 1)
    w = torch.randn(1, 2 * T, 1, 3, dtype=torch.float64)
    _, state = oracle.delta_rule(again, again, w, torch.zeros(1, 2 * T, 1), torch.ones(1, 2 * T, 1), scale=1.0)
    assert torch.allclose(state[0, 0], w[0, T:, 0])


def test_decay_alone_scales_the_state():
    q, k, v, g, _, init = _inputs()
    o, state = oracle.delta_rule(q, k, v, g, torch.zeros_like(g), init_state=init)
    total = g.sum(1).exp()
    assert torch.allclose(state, init * total[..., None, None])
    want = 3 ** -0.5 * torch.einsum("hkv,tk->thv", init[0], q[0, :, 0]) * g[0].cumsum(0).exp()[..., None]
    assert torch.allclose(o[0], want)


def test_packed_sequences_and_lengths_are_separate_rows():
    q, k, v, g, beta, _ = _inputs(T=9)
    lens = [4, 0, 1, 4]
    init = torch.randn(4, 2, 3, 4, dtype=torch.float64)
    o, state = oracle.delta_rule(q, k, v, g, beta, init_state=init, lens=lens, packed=True)
    at = 0
    for n, length in enumerate(lens):
        part = [t[:, at:at + length] for t in (q, k, v, g, beta)]
        want, after = oracle.delta_rule(*part, init_state=init[n:n + 1])
        assert torch.equal(o[:, at:at + length], want) and torch.equal(state[n], after[0])
        at += length
    o, state = oracle.delta_rule(q, k, v, g, beta, lens=[5])
    assert o[0, 5:].abs().max() == 0
    assert torch.equal(state, oracle.delta_rule(*(t[:, :5] for t in (q, k, v, g, beta)))[1])


def test_gradient_against_differences():
    args = [t.requires_grad_() for t in _inputs(T=4)]
    assert torch.autograd.gradcheck(
        lambda q, k, v, g, beta, init: oracle.delta_rule(q, k, v, g, beta, init_state=init), args)


@pytest.mark.parametrize("with_draft", [True, False])
def test_verified_tokens_follow_the_target(with_draft):
    """One draft from q, then verification: the first token's distribution is p,
    whatever q. 40000 trials: a share is off by at most 5 standard deviations,
    5 sqrt(0.25 / 40000) = 0.0125."""
    gen = torch.Generator().manual_seed(1)
    n, V = 40000, 5
    p = torch.tensor([0.1, 0.35, 0.0, 0.3, 0.25])
    q = torch.tensor([0.4, 0.1, 0.2, 0.3, 0.0])
    tokens = torch.multinomial(q, n, replacement=True, generator=gen).view(n, 1)
    draft = q.expand(n, 1, V)
    if not with_draft:
        tokens[:] = 3
        draft = None
    out, taken = oracle.verify_drafts(tokens, p.expand(n, 2, V), draft, torch.rand(n, 1, generator=gen),
                                      torch.rand(n, generator=gen))
    share = torch.bincount(out[:, 0], minlength=V) / n
    assert (share - p).abs().max() < 0.0125 and share[2] == 0
    assert ((out[:, 1] >= 0) == (taken == 1)).all()
