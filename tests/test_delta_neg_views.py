"""Imaginary parts of conjugated tensors: torch keeps them as views whose memory
holds the values with the other sign. The gated delta rule reads the values."""
from __future__ import annotations

import pytest
import torch


def _negated(t):
    """t's values, as a view of memory that holds -t."""
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view


def test_not_eager():
    from ramnet_ops.impl import _delta
    x = torch.rand(3)
    assert _delta.is_eager(x, None, x) and not _delta.is_eager(x, None, _negated(x))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("which", range(6))
def test_inputs(T, which):
    from ramnet_ops import gated_delta_rule
    from test_gpu_delta_rule import DEV, _case
    case = [t.to(DEV) for t in _case(T=T, Dk=16, Dv=1)]
    want = gated_delta_rule(*case[:5], init_state=case[5])
    case[which] = _negated(case[which])
    got = gated_delta_rule(*case[:5], init_state=case[5])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("Dv", [1, 16])
def test_gradients(Dv):
    """The output as the imaginary part of a conjugated tensor: its gradient comes as such a view."""
    from ramnet_ops import gated_delta_rule
    from test_gpu_delta_rule import DEV, _case
    case = [t.to(DEV) for t in _case(T=70, Dk=1, Dv=Dv)]

    def grads(use):
        x = [t.detach().requires_grad_() for t in case]
        o, state = gated_delta_rule(*x[:5], init_state=x[5])
        return torch.autograd.grad([use(o), use(state)], x)

    def plain(y):
        return -(y * y).sum()

    def conjugated(y):
        z = torch.complex(torch.zeros_like(y), y).conj()
        return (z.imag * y.detach()).sum() * 2
    for a, b in zip(grads(conjugated), grads(plain)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("Dv", [1, 16])
def test_gradients_given(Dv):
    from ramnet_ops import gated_delta_rule
    from test_gpu_delta_rule import DEV, _case
    case = [t.to(DEV) for t in _case(T=70, Dk=1, Dv=Dv)]
    d = [torch.randn(1, 70, 1, Dv, device=DEV), torch.randn(1, 1, 1, Dv, device=DEV)]

    def grads(d):
        x = [t.detach().requires_grad_() for t in case]
        return torch.autograd.grad(gated_delta_rule(*x[:5], init_state=x[5]), x, d)
    for a, b in zip(grads([_negated(t) for t in d]), grads(d)):
        assert torch.equal(a, b)
