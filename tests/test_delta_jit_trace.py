"""``torch.jit.trace`` records calls of the gated delta rule and of draft verification."""
from __future__ import annotations

import pytest
import torch


def test_tracing_is_not_eager():
    from ramnet_ops.impl import _delta
    seen = []

    def f(x):
        seen.append(_delta.is_eager(x))
        return x + 1
    x = torch.zeros(2)
    torch.jit.trace(f, (x,), check_trace=False)
    assert seen == [False] and _delta.is_eager(x)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("grad", [False, True])
def test_delta_rule(T, grad):
    from ramnet_ops import gated_delta_rule
    from test_gpu_delta_rule import DEV, _case

    def f(q, k, v, g, beta, init):
        return gated_delta_rule(q, k, v, g, beta, init_state=init)
    first, other = ([t.to(DEV).requires_grad_(grad) for t in _case(T=T, Dk=16, Dv=16, seed=s)] for s in (1, 2))
    traced = torch.jit.trace(f, tuple(first), check_trace=False)
    for case in (first, other):
        for a, b in zip(traced(*case), f(*case)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_verify_drafts():
    from ramnet_ops import verify_drafts

    def case(seed):
        gen = torch.Generator().manual_seed(seed)
        target = torch.softmax(torch.randn(3, 5, 50, generator=gen), -1)
        draft = torch.softmax(torch.randn(3, 4, 50, generator=gen), -1)
        tokens = torch.randint(0, 50, (3, 4), generator=gen)
        return [t.cuda() for t in (tokens, target, draft, torch.rand(3, 4, generator=gen), torch.rand(3, generator=gen))]
    traced = torch.jit.trace(verify_drafts, tuple(case(1)), check_trace=False)
    for x in (case(1), case(2)):
        for a, b in zip(traced(*x), verify_drafts(*x)):
            assert torch.equal(a, b)
