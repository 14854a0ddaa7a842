"""The gated delta rule's state over chunks that mostly decay it, on the GPU.

Where little is written, the state after a chunk and the gradient before it are
the ones given times e^(sum of the chunk's decays), which has to be held to 32
bits of its own size: in a last chunk of fewer than 64 tokens, and in one whose
last keys are zeros, as in any other. Tolerances are those of fp32 arithmetic,
8 sqrt(max(Dk, 64)) 2^-24 in the 2-norm, 8 times that for a decay's gradient.
"""
from __future__ import annotations

import pytest
import torch

from oracle import delta_oracle as oracle
from test_gpu_delta_rule import DEV, _arith, _call, _case, _grads, _rel

pytestmark = pytest.mark.gpu

DTYPES = ["fp32", "fp16", "bf16"]


def _fading(T, dtype, each=0.4, seed=0, **kw):
    """Nothing is written; a token's decay is e^-0.3 to e^-0.5 by default."""
    case = _case(T=T, Hk=1, Hv=2, Dk=40, Dv=48, dtype=dtype, seed=seed, **kw)
    gen = torch.Generator().manual_seed(seed)
    case[3] = -each * (0.75 + 0.5 * torch.rand(case[3].shape, generator=gen))
    case[4] = torch.zeros_like(case[4])
    return case


def _check_state(case, lens=None, packed=False, **kw):
    _, state = _call(case, **kw)
    _, want = oracle.delta_rule(*case[:5], init_state=case[5], lens=lens, packed=packed)
    for n in range(want.shape[0]):
        for h in range(want.shape[1]):
            assert _rel(state[n, h], want[n, h]) <= _arith(40), (n, h, _rel(state[n, h], want[n, h]))


def _check_gradients(case, **kw):
    """Of the state alone (in 32 bits: the others' own rounding would hide the state's)."""
    have, got, want, _ = _grads(case, use=(False, True), **kw)
    for n, a, b in zip(have, got, want):
        if a.dtype == torch.float32:
            tol = _arith(40) * (8 if n == "g" else 1)
            assert _rel(a, b) <= tol, (n, _rel(a, b), tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [9, 40, 63, 64, 100])
def test_state(T, dtype):
    _check_state(_fading(T, dtype, seed=T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [9, 40, 64, 100])
def test_gradients(T, dtype):
    _check_gradients(_fading(T, dtype, seed=T))


@pytest.mark.parametrize("dtype", DTYPES)
def test_last_keys_zero(dtype):
    """As in a padded row: a full chunk whose last keys are zeros."""
    case = _fading(64, dtype, seed=1)
    case[1][:, 50:] = 0
    _check_state(case)
    _check_gradients(case)
    case = _case(T=128, Hk=1, Hv=2, Dk=40, Dv=48, dtype=dtype, seed=2)  # with writes before
    case[1][:, 64:] = 0
    case[3][:, 64:] = -0.25
    _check_state(case)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_packed_and_counted(dtype):
    lens = [40, 0, 1, 100, 64, 30]
    cu = torch.tensor([0] + lens).cumsum(0).to(DEV, torch.int32)
    case = _fading(sum(lens), dtype, N=len(lens), seed=3)
    _check_state(case, lens, packed=True, cu_seqlens=cu)
    _check_gradients(case, kw=dict(cu_seqlens=cu), lens=lens, packed=True)
    lens = [100, 0, 1, 40, 70]
    case = _fading(100, dtype, B=5, seed=4)
    _check_state(case, lens, lengths=torch.tensor(lens, device=DEV))
    _check_gradients(case, kw=dict(lengths=torch.tensor(lens, device=DEV)), lens=lens)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_segments(dtype):
    """A row cut into segments, weak writes, and a last chunk of 12 tokens that decay by e^-1 each."""
    case = _case(T=1100, Hk=1, Hv=2, Dk=40, Dv=48, dtype=dtype, seed=5)
    case[3] = torch.full_like(case[3], -1e-3)
    case[3][:, -12:] = -1
    case[4] = torch.zeros_like(case[4])
    case[4][:, ::97] = 2.0 ** -10
    case[4][:, -12:] = 0
    _check_state(case)
    _check_gradients(case)
