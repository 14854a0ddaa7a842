"""16-bit outputs of the gated delta rule on the GPU are 32-bit results, rounded once.

Compared with the fp64 oracle's values rounded to the type. A result d off its
value before the rounding falls on the other side of a border with probability
d / step, and is a step off then, so the mean square of the difference is at
most the mean of d step. With the arithmetic's bound for d (a relative 2-norm:
8 sqrt(max(Dk, 64)) 2^-24) and a step of at most eps times the value:
sqrt(arith eps), and arith itself on top for values where d is above a step.
A decay's gradient sums terms that cancel: 8 times the arithmetic's. An operand
held in 11 bits is off by 2^-12 or more of it, which bf16 outputs show as 1e-3.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import delta_oracle as oracle
from test_gpu_delta_rule import DEV, _arith, _call, _case, _grads, _rel

pytestmark = pytest.mark.gpu


def _rounded(t, arith):
    return math.sqrt(arith * torch.finfo(t.dtype).eps) + arith


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,Dk,Dv", [(6, 64, 64), (37, 64, 64), (150, 128, 128), (130, 256, 64), (70, 37, 50),
                                     (1100, 64, 48)])
def test_output(dtype, T, Dk, Dv):
    case = _case(T=T, Hk=1, Hv=2, Dk=Dk, Dv=Dv, dtype=dtype, seed=T + Dk)
    o, state = _call(case)
    want, after = oracle.delta_rule(*case[:5], init_state=case[5])
    off = _rel(o, want.to(o.dtype))
    assert off <= _rounded(o, _arith(Dk)), (off, _rounded(o, _arith(Dk)))
    assert _rel(state, after) <= _arith(Dk)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,Dk,Dv", [(37, 64, 64), (130, 128, 128), (70, 37, 50), (70, 256, 64), (1100, 64, 48)])
def test_gradients(dtype, T, Dk, Dv):
    case = _case(T=T, Hk=1, Hv=2, Dk=Dk, Dv=Dv, dtype=dtype, g_dtype=dtype, seed=T + Dk)
    have, got, want, _ = _grads(case)
    for n, a, b in zip(have, got, want):
        arith = (8 if n == "g" else 1) * _arith(Dk)
        if a.dtype == torch.float32:
            assert _rel(a, b) <= arith, n
        else:
            off = _rel(a, b.to(a.dtype))
            assert off <= _rounded(a, arith), (n, off, _rounded(a, arith))


def test_packed_output():
    lens = [5, 0, 70, 200, 1]
    case = _case(T=sum(lens), Hk=1, Hv=2, Dk=64, Dv=64, dtype="bf16", N=len(lens), seed=4)
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    o, _ = _call(case, cu_seqlens=cu)
    want, _ = oracle.delta_rule(*case[:5], init_state=case[5], lens=lens, packed=True)
    assert _rel(o, want.to(o.dtype)) <= _rounded(o, _arith(64))
