"""What the gated delta rule's gradients and precision reach to, on the GPU."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import delta_oracle as oracle
from test_gpu_delta_rule import DEV, _arith, _call, _case, _check, _check_grads

pytestmark = pytest.mark.gpu


def test_second_derivatives_are_refused():
    from ramnet_ops import gated_delta_rule
    x = [t.to(DEV).requires_grad_() for t in _case(T=20, Dk=16, Dv=16)]
    o, _ = gated_delta_rule(*x[:5], init_state=x[5])
    d, = torch.autograd.grad(o.square().sum(), x[0], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()


@pytest.mark.parametrize("size", [4.0, 300.0])
@pytest.mark.parametrize("T", [8, 140])
def test_large_keys(T, size):
    """Keys of norm `size`, with write strengths that keep beta |k|^2 at most 1."""
    for dtype in ("fp32", "bf16"):
        case = _case(T=T, Hk=1, Hv=2, Dk=40, Dv=48, dtype=dtype, seed=12)
        case[1] = (case[1].float() * size).to(case[1].dtype)
        case[4] = (case[4].float() / size ** 2).to(case[4].dtype)
        case[5] = case[5] / size
        _check(case, _call(case))
        if T > 8:
            _check_grads(case)


def test_small_tokens_beside_large_ones():
    """A chunk's products are exact to 2^-39 of the largest value of their column in the
    chunk (two fp16 parts under one scale): a token's own values to 2^-24 down to 2^-15 of
    that. Rounded at random over 64 terms in 8 products, as fp32 arithmetic is:
    8 sqrt(64) (2^-24 |o_t| + 2^-39 |largest|) for each token."""
    T = 64
    case = _case(T=T, Hk=1, Hv=1, Dk=64, Dv=48, seed=13, state=False)
    size = 2.0 ** -torch.linspace(40, 0, T)
    case[2] = case[2] * size[:, None, None]
    o, _ = _call(case)
    want, _ = oracle.delta_rule(*case[:5])
    off = (o.cpu().double() - want).norm(dim=-1).flatten()
    largest = case[2].abs().amax(1).double().norm() / math.sqrt(64)  # scale = Dk ** -0.5
    bound = _arith(64) * want.norm(dim=-1).flatten() + 8 * math.sqrt(64) * 2.0 ** -39 * largest
    assert (off <= bound).all(), (off / bound).max()
